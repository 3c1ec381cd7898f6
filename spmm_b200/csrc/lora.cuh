// Low-rank adapters of many requests beside a sparse product: C (M x N) gets, column by column, the two small factors of
// the column's own adapter.  With a = index[t], D_a (R x K), U_a (M x R) and the scale s_a:
//
//   H[:, t] = s_a D_a X[:, t]        Y[:, t] = base[:, t] + U_a H[:, t]
//   P[:, t] = s_a U_a^T dY[:, t]     dX[:, t] = base[:, t] + D_a^T P[:, t]
//   dD_a = sum_t P[:, t] X[:, t]^T   dU_a = sum_t dY[:, t] H[:, t]^T     (over the columns of adapter a)
//
// A column whose index is not in [0, L) has no adapter: H = P = 0 there and Y = base.
#pragma once

#include <algorithm>
#include <climits>
#include <type_traits>

#include <cooperative_groups.h>

#include "dense.h"

namespace cg = cooperative_groups;

namespace tca {

// Which adapter a column has.
struct Columns {
    const void *index;  // one per column, or NULL: adapter 0 for all
    int wide;           // 64-bit indices
    int L;
    __device__ __forceinline__ int of(long long t) const
    {
        if (!index) return L > 0 ? 0 : -1;
        const long long a = wide ? __ldg((const long long *)index + t) : (long long)__ldg((const int *)index + t);
        return a >= 0 && a < L ? (int)a : -1;
    }
};

// Out = base + F2 S, S = scale F1 In, column by column with the column's adapter.  Forward: F1 = D (stored [r][i]), F2 = U
// (stored [j][r]).  Transposed (dX): F1 = U^T (stored [i][r]), F2 = D^T (stored [r][j]).
struct ApplyParams {
    const void *F1, *F2;
    const float *scale;
    Columns c;
    int R;
    long long n1, n2, N;  // rows of In, rows of Out, columns
    const void *In;
    long long ldin;
    const void *base;  // or NULL
    long long ldbase;
    int basetype;
    void *Out;  // or NULL
    long long ldout;
    int outtype;
    float *S;  // R x N, or NULL
    int vec_in, vec_f1, pair_f2, vec_base, vec_out;  // what alignment allows
    long long per1, per2;  // rows of In and of Out for each block of a cluster
};

// One of the two products of a backward pass: G[a][j, r] = sum over the columns of adapter a of Z[j, t] S[r, t].
struct GradProblem {
    const void *Z;
    long long ldz;
    int z32;  // Z is fp32 (else the factors' type)
    int vec;
    const float *S;
    long long n;
    void *G;  // or NULL: left out
    long long gj, gr;  // strides of G's elements (j, r) within an adapter
    int tiles;
};

struct GradParams {
    GradProblem p[2];
    Columns c;
    int R;
    int vec_s;
    long long N, per;  // columns, columns for each block of a cluster
};

// ------------------------------------------------------------------ instructions
namespace {

__device__ __forceinline__ unsigned smem_addr(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

// 16 bytes from global to shared memory, the bytes past `valid` as zeros.
__device__ __forceinline__ void copy16(void *dst, const void *src, int valid)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <bool TRANS>
__device__ __forceinline__ void load_matrices(unsigned (&d)[4], const void *p)
{
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(smem_addr(p)) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(smem_addr(p)) : "memory");
}

// D (16 x 8) += A (16 x 16) B (16 x 8), 16-bit operands of type T.
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    if (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D (16 x 8) += A (16 x 8) B (8 x 8), TF32 operands.
__device__ __forceinline__ void mma8(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned to_tf32(float x)
{
    unsigned r;
    asm volatile("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}

// x = hi + lo up to 2^-21 |x|, both TF32 values: the upper 10 bits after the point, and what is left.
__device__ __forceinline__ void split_tf32(float x, unsigned &hi, unsigned &lo)
{
    const unsigned b = __float_as_uint(x);
    const bool special = (b & 0x7f800000u) == 0x7f800000u;  // infinities and NaN stay whole
    hi = special ? __float_as_uint(x + x) : b & 0xffffe000u;
    lo = special ? 0u : __float_as_uint(x - __uint_as_float(hi));
}

// x = hi + lo up to 2^-17 |x| (bf16) or 2^-22 (fp16, in its range): two values of type T.  Kept below the type's largest
// value, hi is finite, and an infinity or NaN comes back whole from lo.
template <typename T>
__device__ __forceinline__ void split16(float x, T &hi, T &lo)
{
    constexpr float MOST = std::is_same<T, __half>::value ? 65504.0f : 3.3895313892515355e38f;
    hi = from_float<T>(fminf(fmaxf(x, -MOST), MOST));
    lo = from_float<T>(x - to_float(hi));
}

// Operands of a product as TF32: factors of 16 bits are exact in it; an fp32 operand beside them is rounded (2^-11, a quarter
// of a bf16 result's half step); two fp32 operands are split and multiplied three times (the product of both low parts, 2^-21,
// is left out), which keeps fp32's precision.
template <bool SPLIT> struct Operand;
template <> struct Operand<false> {
    unsigned v;
    __device__ __forceinline__ void set(float x) { v = to_tf32(x); }
};
template <> struct Operand<true> {
    unsigned v, lo;
    __device__ __forceinline__ void set(float x) { split_tf32(x, v, lo); }
};

template <bool SPLIT>
__device__ __forceinline__ void mma8_any(float (&d)[4], const Operand<SPLIT> (&a)[4], const Operand<SPLIT> &b0, const Operand<SPLIT> &b1)
{
    const unsigned hi[4] = {a[0].v, a[1].v, a[2].v, a[3].v};
    if constexpr (SPLIT) {
        const unsigned lo[4] = {a[0].lo, a[1].lo, a[2].lo, a[3].lo};
        mma8(d, lo, b0.v, b1.v);
        mma8(d, hi, b0.lo, b1.lo);
    }
    mma8(d, hi, b0.v, b1.v);
}

// ------------------------------------------------------------------ Out = base + F2 (scale F1 In)
//
// A cluster of up to 8 blocks takes TN columns.  First each block multiplies its part of In's rows: its 8 warps take 16 rows
// (8 in fp32) in turn, each through a ring of its own in shared memory (In's rows and F1's slice by asynchronous copies, no
// barrier in the loop), with all R x TN sums in the warp's registers.  The sums are joined over warps, then over blocks
// through distributed shared memory, in a fixed order, so that S never crosses device memory on its way to the second
// product.  Then each block multiplies its part of Out's rows: a warp takes 16 rows, F2 straight from L2, base read and Out
// written 16 bytes a thread (columns are dealt to the matrix instruction so that a thread's results lie side by side).
// With several adapters among a tile's columns the products run once for each, and a column keeps its own adapter's.
//
// In 16 bits S is held in two parts (split16), so that an fp32 Out is as exact as fp32 sums of exact products; fp16 parts
// are scaled by a power of two for each column, as S may exceed fp16's range.  The tensor cores' legacy form (mma.sync) is
// enough: the kernel moves R / 8 or fewer products a byte and is bound by In, base and Out.
constexpr int APPLY_WARPS = 8;
constexpr int APPLY_THREADS = APPLY_WARPS * 32;

template <typename TF, typename TI, int RT, int TN, bool TRANS>
struct ApplyShape {
    static constexpr bool M16 = sizeof(TF) == 2 && sizeof(TI) == 2;  // 16-bit matrix instructions (else TF32)
    static constexpr bool SPLIT = sizeof(TF) == 4;
    static constexpr int KS = sizeof(TF) == 4 ? 8 : 16;  // rows of In a step
    static constexpr int RP = RT * 16;
    // Row pitches in bytes, padded so that a matrix fragment's rows fall into different banks.
    static constexpr int IN_PITCH = TN * (int)sizeof(TI) + (sizeof(TI) == 4 ? 32 : 16);
    static constexpr int F_ROWS = TRANS ? KS : RP;
    static constexpr int F_COLS = TRANS ? RP : KS;
    static constexpr int F_PITCH = F_COLS * (int)sizeof(TF) + (TRANS && sizeof(TF) == 4 ? 32 : 16);
    static constexpr int STAGE = KS * IN_PITCH + F_ROWS * F_PITCH;
    static constexpr int FIT = 100 * 1024 / (APPLY_WARPS * STAGE);
    static constexpr int STAGES = FIT >= 6 ? 6 : FIT >= 3 ? FIT : 208 * 1024 / (APPLY_WARPS * STAGE) >= 3 ? 3 : 2;
    static constexpr int S_PITCH = TN + 8;  // floats
    static constexpr int S_BYTES = RP * S_PITCH * 4;
    static constexpr int H_PITCH = TN * 2 + 16;  // bytes
    static constexpr int RING = APPLY_WARPS * STAGES * STAGE;
    static constexpr int BYTES = RING > 4 * S_BYTES ? RING : 4 * S_BYTES;
};

template <typename TF, typename TI, int RT, int TN, bool TRANS>
__global__ void __launch_bounds__(APPLY_THREADS) lora_apply(const ApplyParams p)
{
    using Q = ApplyShape<TF, TI, RT, TN, TRANS>;
    constexpr int NB = TN / 8, RP = Q::RP, KS = Q::KS;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int ids[TN], list[TN], count;
    __shared__ float colscale[TN];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2;
    const long long t0 = (long long)(blockIdx.x / ranks) * TN;

    for (int t = threadIdx.x; t < TN; t += APPLY_THREADS) ids[t] = t0 + t < p.N ? p.c.of(t0 + t) : -1;
    __syncthreads();
    if (warp == 0) {  // the tile's adapters, in the order of their first columns
        int n = 0;
        for (int b = 0; b < TN; b += 32) {
            const int t = b + lane;
            bool first = t < TN && ids[t] >= 0;
            for (int s = 0; first && s < t; ++s) first = ids[s] != ids[t];
            const unsigned m = __ballot_sync(~0u, first);
            if (first) list[n + __popc(m & ((1u << lane) - 1))] = ids[t];
            n += __popc(m);
        }
        if (lane == 0) count = n;
    }
    __syncthreads();
    const int nd = count;

    // ---- S: this block's rows of In
    float acc[RT][NB][4];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][b][e] = 0.0f;
    const long long i_begin = min(p.n1, rank * p.per1), i_end = min(p.n1, i_begin + p.per1);
    const int steps = (int)((i_end - i_begin + KS - 1) / KS);
    const int mine = steps > warp ? (steps - warp + APPLY_WARPS - 1) / APPLY_WARPS : 0;
    const int items = mine * nd;
    unsigned char *ring = smem + warp * (Q::STAGES * Q::STAGE);

    auto fill = [&](int slot, int step, int a) {
        unsigned char *in = ring + slot * Q::STAGE, *f = in + KS * Q::IN_PITCH;
        const long long i0 = i_begin + (long long)(warp + step * APPLY_WARPS) * KS;
        const TI *src = (const TI *)p.In + i0 * p.ldin + t0;
        if (p.vec_in) {
            constexpr int PER = 16 / (int)sizeof(TI), CH = TN / PER;
            for (int k = lane; k < KS * CH; k += 32) {
                const int r = k / CH, c = (k - r * CH) * PER;
                const long long left = i0 + r < i_end ? p.N - t0 - c : 0;
                const int valid = left <= 0 ? 0 : left >= PER ? 16 : (int)left * (int)sizeof(TI);
                copy16(in + r * Q::IN_PITCH + c * sizeof(TI), valid ? src + r * p.ldin + c : (const TI *)p.In, valid);
            }
        } else {
            for (int k = lane; k < KS * TN; k += 32) {
                const int r = k / TN, c = k - r * TN;
                TI v = from_float<TI>(0.0f);
                if (i0 + r < i_end && t0 + c < p.N) v = src[r * p.ldin + c];
                *(TI *)(in + r * Q::IN_PITCH + c * sizeof(TI)) = v;
            }
        }
        const TF *F = (const TF *)p.F1 + (long long)a * p.R * p.n1;
        const long long rows_left = i_end - i0;
        if (p.vec_f1) {
            constexpr int PER = 16 / (int)sizeof(TF), CH = Q::F_COLS / PER;
            for (int k = lane; k < Q::F_ROWS * CH; k += 32) {
                const int r = k / CH, c = (k - r * CH) * PER;
                const long long left = TRANS ? (r < rows_left ? p.R - c : 0) : (r < p.R ? rows_left - c : 0);
                const int valid = left <= 0 ? 0 : left >= PER ? 16 : (int)left * (int)sizeof(TF);
                const TF *s = TRANS ? F + (i0 + r) * p.R + c : F + (long long)r * p.n1 + i0 + c;
                copy16(f + r * Q::F_PITCH + c * sizeof(TF), valid ? s : (const TF *)p.F1, valid);
            }
        } else {
            for (int k = lane; k < Q::F_ROWS * Q::F_COLS; k += 32) {
                const int r = k / Q::F_COLS, c = k - r * Q::F_COLS;
                TF v = from_float<TF>(0.0f);
                if (TRANS ? (r < rows_left && c < p.R) : (r < p.R && c < rows_left))
                    v = TRANS ? F[(i0 + r) * p.R + c] : F[(long long)r * p.n1 + i0 + c];
                *(TF *)(f + r * Q::F_PITCH + c * sizeof(TF)) = v;
            }
        }
    };

    int next_step = 0, next_d = 0, filled = 0;
    auto fill_next = [&]() {
        if (filled < items) {
            fill(filled % Q::STAGES, next_step, list[next_d]);
            if (++next_d == nd) {
                next_d = 0;
                ++next_step;
            }
            ++filled;
        }
        copy_commit();
    };
#pragma unroll
    for (int s = 0; s < Q::STAGES - 1; ++s) fill_next();
    int d = 0;
    for (int it = 0; it < items; ++it) {
        copy_wait<Q::STAGES - 2>();
        __syncwarp();
        const unsigned char *in = ring + (it % Q::STAGES) * Q::STAGE, *f = in + KS * Q::IN_PITCH;
        const int a = list[d];
        // Which blocks of 8 columns hold columns of adapter a, and which others beside them.
        unsigned some = ~0u, mixed = 0u;
        if (nd > 1) {
            some = 0u;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int o = ids[b * 8 + (lane & 7)];
                if (__any_sync(~0u, o == a)) some |= 1u << b;
                if (__any_sync(~0u, o != a && o >= 0)) mixed |= 1u << b;
            }
        }
        // acc += part, or in a mixed block only for adapter a's columns.
        auto add = [&](auto &&product) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!(some >> b & 1)) continue;
#pragma unroll
                for (int m = 0; m < RT; ++m) {
                    if (!(mixed >> b & 1)) {
                        product(m, b, acc[m][b]);
                    } else {
                        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        product(m, b, part);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (ids[b * 8 + 2 * q + (e & 1)] == a) acc[m][b][e] += part[e];
                    }
                }
            }
        };
        if constexpr (Q::M16) {
            unsigned A[RT][4], B[NB][2];
#pragma unroll
            for (int m = 0; m < RT; ++m)
                load_matrices<TRANS>(A[m], TRANS ? f + ((lane & 7) + (lane >> 4) * 8) * Q::F_PITCH + (m * 16 + (lane >> 3 & 1) * 8) * 2
                                                 : f + (m * 16 + (lane & 15)) * Q::F_PITCH + (lane >> 4) * 16);
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                unsigned t[4];
                load_matrices<true>(t, in + (lane & 15) * Q::IN_PITCH + (b + (lane >> 4)) * 16);
                B[b][0] = t[0];
                B[b][1] = t[1];
                B[b + 1][0] = t[2];
                B[b + 1][1] = t[3];
            }
            add([&](int m, int b, float (&to)[4]) { mma16<TF>(to, A[m], B[b][0], B[b][1]); });
        } else {
#pragma unroll
            for (int k = 0; k < KS; k += 8) {
                Operand<Q::SPLIT> A[RT][4];
#pragma unroll
                for (int m = 0; m < RT; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = m * 16 + g + (e & 1) * 8, i = k + q + (e >> 1) * 4;
                        A[m][e].set(to_float(*(const TF *)(TRANS ? f + i * Q::F_PITCH + r * sizeof(TF) : f + r * Q::F_PITCH + i * sizeof(TF))));
                    }
                Operand<Q::SPLIT> B[2];
                int have = -1;
                add([&](int m, int b, float (&to)[4]) {
                    if (have != b) {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            B[e].set(to_float(*(const TI *)(in + (k + q + e * 4) * Q::IN_PITCH + (b * 8 + g) * sizeof(TI))));
                        have = b;
                    }
                    mma8_any<Q::SPLIT>(to, A[m], B[0], B[1]);
                });
            }
        }
        if (++d == nd) d = 0;
        __syncwarp();
        fill_next();
    }
    copy_wait<0>();
    __syncthreads();

    // ---- S joined over the warps: 4 to 7 leave theirs, 0 to 3 add them to their own, all threads add those four
    float *slot = (float *)smem;
    constexpr int SLOT = Q::S_BYTES / 4, PITCH = Q::S_PITCH;
    auto frag = [&](float *s, bool add) {
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float2 *to = (float2 *)(s + (m * 16 + g + h * 8) * PITCH + b * 8 + 2 * q);
                    float2 v = make_float2(acc[m][b][2 * h], acc[m][b][2 * h + 1]);
                    if (add) {
                        const float2 o = *to;
                        v.x += o.x;
                        v.y += o.y;
                    }
                    *to = v;
                }
    };
    if (warp >= 4) frag(slot + (warp - 4) * SLOT, false);
    __syncthreads();
    if (warp < 4) frag(slot + warp * SLOT, true);
    __syncthreads();
    for (int i = threadIdx.x; i < RP * TN; i += APPLY_THREADS) {
        float *s = slot + i / TN * PITCH + i % TN;
        s[0] = (s[0] + s[SLOT]) + (s[2 * SLOT] + s[3 * SLOT]);
    }
    cluster.sync();

    // ---- S joined over the blocks: each takes TN / ranks columns, scales them and gives them to all
    float *Hf = slot + SLOT;
    const int own = TN / ranks;
    for (int cgroup = warp; cgroup * 4 < own; cgroup += APPLY_WARPS) {
        const int c = rank * own + cgroup * 4 + q;
        const bool in = cgroup * 4 + q < own;
        float most = 0.0f;
        const int a = in ? ids[c] : -1;
        const float s = a >= 0 ? (p.scale ? __ldg(p.scale + a) : 1.0f) : 0.0f;
        for (int r = g; r < RP; r += 8) {
            float v = 0.0f;
            if (a >= 0) {
                for (int k = 0; k < ranks; ++k) v += cluster.map_shared_rank(slot, k)[r * PITCH + c];
                v *= s;
            }
            if (in && p.S && r < p.R && t0 + c < p.N) p.S[(long long)r * p.N + t0 + c] = v;
            if (std::is_same<TF, __half>::value) {
                if (in) Hf[r * PITCH + c] = v;
                most = fmaxf(most, fabsf(v));
            } else if (in) {
                for (int k = 0; k < ranks; ++k) cluster.map_shared_rank(Hf, k)[r * PITCH + c] = v;
            }
        }
        if (std::is_same<TF, __half>::value) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
            // The column's largest value goes to [2^13, 2^14); zeros and infinities stay.
            const int e = (__float_as_int(most) >> 23) - 127;
            const int shift = e == -127 || e == 128 ? 0 : max(-100, min(100, e - 13));
            const float down = __int_as_float((127 - shift) << 23), up = __int_as_float((127 + shift) << 23);
            if (in) {
                for (int r = g; r < RP; r += 8) {
                    const float v = Hf[r * PITCH + c] * down;
                    for (int k = 0; k < ranks; ++k) cluster.map_shared_rank(Hf, k)[r * PITCH + c] = v;
                }
                if (g == 0)
                    for (int k = 0; k < ranks; ++k) cluster.map_shared_rank(colscale, k)[c] = up;
            }
        }
    }
    cluster.sync();
    if (!p.Out) return;

    // ---- S as the second product's operand.  Column c of a pair of 8-column blocks holds the tile's column
    // 4 (c % 8 / 2) + 2 (c / 8) + c % 2, so that a thread's results of the pair are four neighbours.
    unsigned char *hi = (unsigned char *)(slot + 2 * SLOT), *lo = (unsigned char *)(slot + 3 * SLOT);
    if constexpr (sizeof(TF) == 2) {
        for (int i = threadIdx.x; i < RP * TN; i += APPLY_THREADS) {
            const int r = i / TN, c = i % TN, t = (c & ~15) + 4 * (c >> 1 & 3) + 2 * (c >> 3 & 1) + (c & 1);
            TF h, l;
            split16<TF>(Hf[r * PITCH + t], h, l);
            *(TF *)(hi + r * Q::H_PITCH + c * 2) = h;
            *(TF *)(lo + r * Q::H_PITCH + c * 2) = l;
        }
        __syncthreads();
    }

    // ---- Out: this block's rows
    const long long j_begin = min(p.n2, rank * p.per2), j_end = min(p.n2, j_begin + p.per2);
    constexpr int PAIRS = TN / 16;
    constexpr int KT = sizeof(TF) == 2 ? RT : RT * 2;  // matrix instructions along r
    for (long long j0 = j_begin + warp * 16; j0 < j_end; j0 += APPLY_WARPS * 16) {
        float4 old[PAIRS][2];
#pragma unroll
        for (int b = 0; b < PAIRS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long j = j0 + g + h * 8, t = t0 + b * 16 + 4 * q;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (p.base && j < j_end && t < p.N) {
                    const long long at = j * p.ldbase + t;
                    if (p.vec_base && t + 3 < p.N) {
                        if (p.basetype == 0) {
                            v = *(const float4 *)((const float *)p.base + at);
                        } else {
                            const uint2 w = *(const uint2 *)((const unsigned short *)p.base + at);
                            const unsigned short u[4] = {(unsigned short)w.x, (unsigned short)(w.x >> 16), (unsigned short)w.y,
                                                         (unsigned short)(w.y >> 16)};
                            float x[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                x[e] = p.basetype == 1 ? __half2float(__ushort_as_half(u[e])) : __bfloat162float(__ushort_as_bfloat16(u[e]));
                            v = make_float4(x[0], x[1], x[2], x[3]);
                        }
                    } else {
                        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (t + e < p.N) {
                                if (p.basetype == 0)
                                    x[e] = ((const float *)p.base)[at + e];
                                else if (p.basetype == 1)
                                    x[e] = __half2float(__ushort_as_half(((const unsigned short *)p.base)[at + e]));
                                else
                                    x[e] = __bfloat162float(__ushort_as_bfloat16(((const unsigned short *)p.base)[at + e]));
                            }
                        v = make_float4(x[0], x[1], x[2], x[3]);
                    }
                }
                old[b][h] = v;
            }
        unsigned A16[sizeof(TF) == 2 ? RT : 1][4];
        Operand<true> A32[sizeof(TF) == 4 ? KT : 1][4];
        auto load_f2 = [&](int a) {
            const TF *F = (const TF *)p.F2 + (long long)a * p.R * p.n2;
            if constexpr (sizeof(TF) == 2) {
                const unsigned short *f = (const unsigned short *)F;
#pragma unroll
                for (int k = 0; k < RT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const long long j = j0 + g + (e & 1) * 8;
                        const int r = k * 16 + 2 * q + (e >> 1) * 8;
                        unsigned v = 0u;
                        if (j < j_end && r < p.R) {
                            if (!TRANS && p.pair_f2) {
                                v = __ldg((const unsigned *)(f + j * p.R + r));
                            } else {
                                v = __ldg(TRANS ? f + (long long)r * p.n2 + j : f + j * p.R + r);
                                if (r + 1 < p.R) v |= (unsigned)__ldg(TRANS ? f + (long long)(r + 1) * p.n2 + j : f + j * p.R + r + 1) << 16;
                            }
                        }
                        A16[k][e] = v;
                    }
            } else {
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const long long j = j0 + g + (e & 1) * 8;
                        const int r = k * 8 + q + (e >> 1) * 4;
                        float v = 0.0f;
                        if (j < j_end && r < p.R) v = __ldg((const float *)F + (TRANS ? (long long)r * p.n2 + j : j * p.R + r));
                        A32[k][e].set(v);
                    }
            }
        };
        if (nd == 1) load_f2(list[0]);
#pragma unroll
        for (int b = 0; b < PAIRS; ++b) {
            int id[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) id[e] = ids[b * 16 + 4 * q + e];
            float sum[2][4] = {};  // [block of the pair][e]: rows g, g + 8; columns 4q + 2 block + (e & 1)
            for (int k = 0; k < nd; ++k) {
                const int a = list[k];
                if (nd > 1) {
                    if (!__any_sync(~0u, id[0] == a || id[1] == a || id[2] == a || id[3] == a)) continue;
                    load_f2(a);
                }
                float part[2][4] = {};
                if constexpr (sizeof(TF) == 2) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        unsigned B[4];
                        const int at = (r * 16 + (lane & 15)) * Q::H_PITCH + (b * 2 + (lane >> 4)) * 16;
                        load_matrices<true>(B, lo + at);
                        mma16<TF>(part[0], A16[r], B[0], B[1]);
                        mma16<TF>(part[1], A16[r], B[2], B[3]);
                        load_matrices<true>(B, hi + at);
                        mma16<TF>(part[0], A16[r], B[0], B[1]);
                        mma16<TF>(part[1], A16[r], B[2], B[3]);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < KT; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int t = b * 16 + 4 * (g >> 1) + 2 * h + (g & 1);
                            Operand<true> B[2];
                            B[0].set(Hf[(r * 8 + q) * PITCH + t]);
                            B[1].set(Hf[(r * 8 + q + 4) * PITCH + t]);
                            mma8_any<true>(part[h], A32[r], B[0], B[1]);
                        }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (id[2 * h + (e & 1)] == a) sum[h][e] = part[h][e];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long j = j0 + g + h * 8, t = t0 + b * 16 + 4 * q;
                if (j >= j_end || t >= p.N) continue;
                const float x[4] = {old[b][h].x, old[b][h].y, old[b][h].z, old[b][h].w};
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = sum[e >> 1][2 * h + (e & 1)];
                    if (std::is_same<TF, __half>::value) v *= colscale[b * 16 + 4 * q + e];
                    y[e] = id[e] >= 0 ? x[e] + v : x[e];
                }
                const long long at = j * p.ldout + t;
                if (p.vec_out && t + 3 < p.N) {
                    if (p.outtype == 0) {
                        *(float4 *)((float *)p.Out + at) = make_float4(y[0], y[1], y[2], y[3]);
                    } else {
                        unsigned short u[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            u[e] = p.outtype == 1 ? __half_as_ushort(__float2half_rn(y[e])) : __bfloat16_as_ushort(__float2bfloat16_rn(y[e]));
                        *(uint2 *)((unsigned short *)p.Out + at) =
                            make_uint2(u[0] | (unsigned)u[1] << 16, u[2] | (unsigned)u[3] << 16);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (t + e < p.N) store_as(p.Out, p.outtype, at + e, y[e]);
                }
            }
        }
    }
}

// ------------------------------------------------------------------ gradients of the factors
//
// A cluster of up to 8 blocks takes 128 rows j of Z and one adapter; its blocks share the columns.  A block goes over the
// chunks of 32 columns that hold any of the adapter's, Z's and S's chunks through a ring in shared memory; a warp takes 16
// rows and all R of S.  Columns of other adapters count as zeros in both operands (an infinity there meets a zero nowhere).
// The blocks' sums are joined through distributed shared memory in a fixed order.  Both products of a backward pass are one
// launch.
constexpr int GRAD_ROWS = 128;
constexpr int GRAD_CHUNK = 32;
constexpr int GRAD_SCAN = 64;  // chunks looked over at once

template <int RT>
struct GradShape {
    static constexpr int RP = RT * 16;
    static constexpr int PITCH = GRAD_CHUNK * 4 + 16;  // bytes of a chunk's row (16-bit rows use a part)
    static constexpr int STAGE = (GRAD_ROWS + RP) * PITCH + GRAD_CHUNK * 4;
    static constexpr int STAGES = RT <= 4 ? 4 : 3;
    static constexpr int SUM_PITCH = RP + 4;  // floats
    static constexpr int SUM = GRAD_ROWS * SUM_PITCH * 4;
    static constexpr int BYTES = STAGE * STAGES > SUM ? STAGE * STAGES : SUM;
};

template <typename TF, typename TZ, int RT>
__device__ __forceinline__ void grad_block(const GradProblem &p, const GradParams &w, long long j0, int a, unsigned char *smem,
                                           float (&acc)[RT * 2][4])
{
    using Q = GradShape<RT>;
    constexpr bool SPLIT = sizeof(TF) == 4;
    __shared__ unsigned char flags[GRAD_SCAN];
    __shared__ unsigned char list[GRAD_SCAN];
    __shared__ int count;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2;
    const cg::cluster_group cluster = cg::this_cluster();
    const long long t_begin = min(w.N, cluster.block_rank() * w.per), t_end = min(w.N, t_begin + w.per);

    auto fill = [&](int slot, long long t0) {
        unsigned char *z = smem + slot * Q::STAGE, *s = z + GRAD_ROWS * Q::PITCH;
        int *ids = (int *)(s + Q::RP * Q::PITCH);
        if (p.vec) {
            constexpr int PER = 16 / (int)sizeof(TZ), CH = GRAD_CHUNK / PER;
            for (int k = threadIdx.x; k < GRAD_ROWS * CH; k += 256) {
                const int r = k / CH, c = (k - r * CH) * PER;
                const long long left = j0 + r < p.n ? t_end - t0 - c : 0;
                const int valid = left <= 0 ? 0 : left >= PER ? 16 : (int)left * (int)sizeof(TZ);
                copy16(z + r * Q::PITCH + c * sizeof(TZ), valid ? (const TZ *)p.Z + (j0 + r) * p.ldz + t0 + c : (const TZ *)p.Z, valid);
            }
        } else {
            for (int k = threadIdx.x; k < GRAD_ROWS * GRAD_CHUNK; k += 256) {
                const int r = k / GRAD_CHUNK, c = k % GRAD_CHUNK;
                TZ v = from_float<TZ>(0.0f);
                if (j0 + r < p.n && t0 + c < t_end) v = ((const TZ *)p.Z)[(j0 + r) * p.ldz + t0 + c];
                *(TZ *)(z + r * Q::PITCH + c * sizeof(TZ)) = v;
            }
        }
        if (w.vec_s) {
            constexpr int CH = GRAD_CHUNK / 4;
            for (int k = threadIdx.x; k < Q::RP * CH; k += 256) {
                const int r = k / CH, c = (k - r * CH) * 4;
                const long long left = r < w.R ? t_end - t0 - c : 0;
                const int valid = left <= 0 ? 0 : left >= 4 ? 16 : (int)left * 4;
                copy16(s + r * Q::PITCH + c * 4, valid ? p.S + (long long)r * w.N + t0 + c : p.S, valid);
            }
        } else {
            for (int k = threadIdx.x; k < Q::RP * GRAD_CHUNK; k += 256) {
                const int r = k / GRAD_CHUNK, c = k % GRAD_CHUNK;
                *(float *)(s + r * Q::PITCH + c * 4) = r < w.R && t0 + c < t_end ? p.S[(long long)r * w.N + t0 + c] : 0.0f;
            }
        }
        if (threadIdx.x < GRAD_CHUNK) ids[threadIdx.x] = t0 + threadIdx.x < t_end ? w.c.of(t0 + threadIdx.x) : a;
    };

    for (long long scan = t_begin; scan < t_end; scan += GRAD_SCAN * GRAD_CHUNK) {
        __syncthreads();
        for (int k = warp; k < GRAD_SCAN; k += 8) {
            const long long t = scan + k * GRAD_CHUNK + lane;
            const int id = t < t_end ? w.c.of(t) : -1;
            const bool any = __any_sync(~0u, id == a), other = __any_sync(~0u, t < t_end && id != a);
            if (lane == 0) flags[k] = any ? (other ? 2 : 1) : 0;
        }
        __syncthreads();
        if (warp == 0) {
            int n = 0;
            for (int k = lane; k < GRAD_SCAN; k += 32) {
                const unsigned m = __ballot_sync(~0u, flags[k] != 0);
                if (flags[k]) list[n + __popc(m & ((1u << lane) - 1))] = (unsigned char)k;
                n += __popc(m);
            }
            if (lane == 0) count = n;
        }
        __syncthreads();
        const int chunks = count;
        auto fill_at = [&](int i) {
            if (i < chunks) fill(i % Q::STAGES, scan + list[i] * GRAD_CHUNK);
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < Q::STAGES - 1; ++i) fill_at(i);
        for (int i = 0; i < chunks; ++i) {
            copy_wait<Q::STAGES - 2>();
            __syncthreads();
            fill_at(i + Q::STAGES - 1);
            const unsigned char *z = smem + (i % Q::STAGES) * Q::STAGE + warp * 16 * Q::PITCH;
            const unsigned char *s = smem + (i % Q::STAGES) * Q::STAGE + GRAD_ROWS * Q::PITCH;
            const int *ids = (const int *)(s + Q::RP * Q::PITCH);
            const bool mixed = flags[list[i]] == 2;
#pragma unroll
            for (int k = 0; k < GRAD_CHUNK; k += 8) {
                Operand<SPLIT> A[4];
                const bool in[2] = {!mixed || ids[k + q] == a, !mixed || ids[k + q + 4] == a};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = to_float(*(const TZ *)(z + (g + (e & 1) * 8) * Q::PITCH + (k + q + (e >> 1) * 4) * sizeof(TZ)));
                    A[e].set(in[e >> 1] ? v : 0.0f);
                }
#pragma unroll
                for (int b = 0; b < RT * 2; ++b) {
                    Operand<SPLIT> B[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = *(const float *)(s + (b * 8 + g) * Q::PITCH + (k + q + e * 4) * 4);
                        B[e].set(in[e] ? v : 0.0f);
                    }
                    mma8_any<SPLIT>(acc[b], A, B[0], B[1]);
                }
            }
        }
        copy_wait<0>();
    }
}

template <typename TF, int RT>
__global__ void __launch_bounds__(256) lora_grad(const GradParams w)
{
    using Q = GradShape<RT>;
    extern __shared__ __align__(16) unsigned char smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2;
    const int tile = blockIdx.x / ranks;
    const bool second = tile >= w.p[0].tiles;
    const GradProblem p = second ? w.p[1] : w.p[0];
    const long long j0 = (long long)(second ? tile - w.p[0].tiles : tile) * GRAD_ROWS;
    for (int a = blockIdx.y; a < w.c.L; a += gridDim.y) {
        float acc[RT * 2][4];
#pragma unroll
        for (int b = 0; b < RT * 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[b][e] = 0.0f;
        if (p.z32)
            grad_block<TF, float, RT>(p, w, j0, a, smem, acc);
        else
            grad_block<TF, TF, RT>(p, w, j0, a, smem, acc);
        __syncthreads();
        float *sum = (float *)smem;
#pragma unroll
        for (int b = 0; b < RT * 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[(warp * 16 + g + (e >> 1) * 8) * Q::SUM_PITCH + b * 8 + 2 * q + (e & 1)] = acc[b][e];
        cluster.sync();
        const int own = GRAD_ROWS / ranks;
        TF *G = (TF *)p.G + (long long)a * p.n * w.R;
        for (int i = threadIdx.x; i < own * w.R; i += 256) {
            // Neighbouring threads write neighbouring elements.
            const int r = p.gr == 1 ? i % w.R : i / own, j = rank * own + (p.gr == 1 ? i / w.R : i % own);
            if (j0 + j >= p.n) continue;
            float v = 0.0f;
            for (int k = 0; k < ranks; ++k) v += cluster.map_shared_rank(sum, k)[j * Q::SUM_PITCH + r];
            G[(j0 + j) * p.gj + r * p.gr] = from_float<TF>(v);
        }
        cluster.sync();
    }
}

// ------------------------------------------------------------------ launches
template <typename... Args>
tcaspmm_status launch_cluster(const char *what, void (*kernel)(Args...), dim3 grid, int threads, int ranks, int shared, cudaStream_t st,
                              Args... args)
{
    if (shared > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (e != cudaSuccess) return cuda_fail(e, what);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? TCASPMM_OK : cuda_fail(e, what);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Calls f with the number of 16-row tiles that hold R, as a compile-time power of two.
template <typename F>
tcaspmm_status with_rank(int R, F &&f)
{
    if (R <= 16) return f(std::integral_constant<int, 1>{});
    if (R <= 32) return f(std::integral_constant<int, 2>{});
    if (R <= 64) return f(std::integral_constant<int, 4>{});
    if (R <= 128) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 16>{});
}

// Columns of a tile: a warp's sums (RT x TN / 8 x 4 registers a thread) take at most 128 registers.
constexpr int tile_columns(int rt) { return rt <= 4 ? 64 : rt == 8 ? 32 : 16; }

template <typename TF, typename TI, bool TRANS>
tcaspmm_status apply(ApplyParams p, int sms, cudaStream_t st)
{
    return with_rank(p.R, [&](auto rt) {
        constexpr int RT = rt.value, TN = tile_columns(RT);
        using Q = ApplyShape<TF, TI, RT, TN, TRANS>;
        const long long tiles = ceil_div(p.N, TN);
        int ranks = 1;  // idle SMs take a share, while a warp has a step to do
        while (ranks < 8 && tiles * ranks < 2 * sms && std::max(p.n1, p.n2) > (long long)ranks * APPLY_WARPS * 16) ranks *= 2;
        p.per1 = ceil_div(ceil_div(p.n1, ranks), Q::KS) * Q::KS;
        p.per2 = ceil_div(ceil_div(p.n2, ranks), 16) * 16;
        if (tiles * ranks > INT_MAX) return fail(TCASPMM_ERR_UNSUPPORTED, "lora: too many columns");
        return launch_cluster("lora launch", lora_apply<TF, TI, RT, TN, TRANS>, dim3((unsigned)(tiles * ranks)), APPLY_THREADS, ranks,
                              Q::BYTES, st, p);
    });
}

template <typename TF>
tcaspmm_status grads(GradParams w, int sms, cudaStream_t st)
{
    return with_rank(w.R, [&](auto rt) {
        constexpr int RT = rt.value;
        for (GradProblem &p : w.p) p.tiles = p.G ? (int)ceil_div(p.n, GRAD_ROWS) : 0;
        const long long tiles = (long long)w.p[0].tiles + w.p[1].tiles;
        if (tiles == 0 || w.c.L == 0) return TCASPMM_OK;
        int ranks = 1;
        while (ranks < 8 && tiles * ranks < 2 * sms && w.N > (long long)ranks * 2 * GRAD_CHUNK) ranks *= 2;
        w.per = ceil_div(ceil_div(w.N, ranks), GRAD_CHUNK) * GRAD_CHUNK;
        if (tiles * ranks > INT_MAX) return fail(TCASPMM_ERR_UNSUPPORTED, "lora_backward: too many rows");
        return launch_cluster("lora_backward launch", lora_grad<TF, RT>, dim3((unsigned)(tiles * ranks), (unsigned)std::min(w.c.L, 65535)),
                              256, ranks, GradShape<RT>::BYTES, st, w);
    });
}

}  // namespace
}  // namespace tca
