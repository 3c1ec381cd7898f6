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
#include <atomic>
#include <cfloat>
#include <climits>
#include <cstring>
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
    // Those of columns t, t + step, ... below `end` (-2 past it), all loads in flight at once.
    template <int COUNT>
    __device__ __forceinline__ void of(long long t, long long step, long long end, int (&a)[COUNT]) const
    {
        if (index && wide) {
            long long raw[COUNT];
#pragma unroll
            for (int k = 0; k < COUNT; ++k) raw[k] = t + k * step < end ? __ldg((const long long *)index + t + k * step) : -1;
#pragma unroll
            for (int k = 0; k < COUNT; ++k) a[k] = raw[k] >= 0 && raw[k] < L ? (int)raw[k] : -1;
        } else if (index) {
#pragma unroll
            for (int k = 0; k < COUNT; ++k) a[k] = t + k * step < end ? __ldg((const int *)index + t + k * step) : -1;
#pragma unroll
            for (int k = 0; k < COUNT; ++k) a[k] = a[k] < L ? max(a[k], -1) : -1;
        } else {
#pragma unroll
            for (int k = 0; k < COUNT; ++k) a[k] = L > 0 ? 0 : -1;
        }
#pragma unroll
        for (int k = 0; k < COUNT; ++k)
            if (t + k * step >= end) a[k] = -2;
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
    void *hidden;  // S (Hidden)
    int vec_in, vec_f1, vec_f2, vec_base, vec_out;  // what alignment allows
    int word_in, word_f1, word_f2;                  // rows start on 4 bytes
    long long per1;  // rows of In for each block of a cluster
    int chunks;      // of EXP_ROWS rows of Out for each block
};

// S in device memory between the kernels, rows of `pitch` columns (64 or a multiple, so that every row is aligned): fp32 for
// the gradients and for fp32 factors, and for 16-bit factors parts of their type whose sum it is: two of fp16 (22 bits; they
// are scaled: a column's, times its colscale, is S), three of bf16 (24 bits).  The parts' columns are dealt out within each 16 (place) so that the
// second product's matrix instructions give a thread four neighbours.  Columns past N hold nothing that counts.
struct Hidden {
    long long pitch, rows;
    unsigned char *p;
    __host__ __device__ static long long pitch_of(long long N) { return (N + 63) / 64 * 64; }
    __host__ static size_t bytes(long long R, long long N, int type)
    {
        return (size_t)pitch_of(N) * (R * (type == 0 ? 4 : type == 1 ? 8 : 10) + (type == 1 ? 4 : 0));
    }
    __host__ __device__ Hidden(void *at, long long R, long long N) : pitch(pitch_of(N)), rows(R), p((unsigned char *)at) {}
    // Where column c of the parts lies: c = 4 i + 2 b + e of each 16 is column 2 i + e of block b of 8.
    __host__ __device__ static int place(int c) { return (c & ~15) + 8 * (c >> 1 & 1) + 2 * (c >> 2 & 3) + (c & 1); }
    __host__ __device__ float *s() const { return (float *)p; }
    template <typename T> __device__ T *part(int i) const { return (T *)(p + pitch * rows * (4 + 2 * i)); }  // the largest first
    __device__ float *colscale() const { return (float *)(p + pitch * rows * 8); }
};

// One of the two products of a backward pass: G[a][j, r] = sum over the columns of adapter a of Z[j, t] S[r, t].
struct GradProblem {
    const void *Z;
    long long ldz;
    int z32;  // Z is fp32 (else the factors' type)
    int vec, word;  // what alignment allows: 16 bytes, 4 bytes
    const float *S;  // rows of Hidden's pitch
    long long n;
    void *G;  // or NULL: left out
    long long gj, gr;  // strides of G's elements (j, r) within an adapter
    int tiles;
};

struct GradParams {
    GradProblem p[2];
    Columns c;
    int R;
    long long N;
};

// ------------------------------------------------------------------ instructions
namespace {

__device__ __forceinline__ unsigned smem_addr(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

// 16 bytes from global to shared memory, the bytes past `valid` as zeros.
__device__ __forceinline__ void copy16(void *dst, const void *src, int valid)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid) : "memory");
}
// 8 bytes, all of them or (valid 0) zeros.
__device__ __forceinline__ void copy8(void *dst, const void *src, int valid)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid) : "memory");
}
// 4 bytes, those past `valid` as zeros.
__device__ __forceinline__ void copy4(void *dst, const void *src, int valid)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid) : "memory");
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
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D (16 x 8) += A (16 x 8) B (8 x 8), TF32 operands.
__device__ __forceinline__ void mma8(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A 16-bit element of type code 1 (fp16) or 2 (bf16).
__device__ __forceinline__ float as_float(unsigned bits, int type)
{
    return type == 1 ? __half2float(__ushort_as_half((unsigned short)bits)) : __bfloat162float(__ushort_as_bfloat16((unsigned short)bits));
}

// x as a sum of PARTS values of type T: all 24 bits of it in three bf16 parts, 22 in two fp16 ones.  The parts have x's sign and
// none is zero unless x is (a first part that would leave nothing gives up its last bit), so that an infinite factor times each
// of them is what it is times x.  An infinity or NaN is the last part, behind ones.
template <typename T> constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 3;
template <typename T>
__device__ __forceinline__ void split16(float x, T (&part)[PARTS<T>])
{
    const bool finite = fabsf(x) <= FLT_MAX;
#pragma unroll
    for (int i = 0; i + 1 < PARTS<T>; ++i) {
        unsigned short bits;
        if constexpr (std::is_same<T, __half>::value)
            bits = __half_as_ushort(__float2half_rz(x));
        else
            bits = (unsigned short)(__float_as_uint(x) >> 16);
        const auto value = [&] { return as_float(bits, std::is_same<T, __half>::value ? 1 : 2); };
        if (!finite)
            bits = (unsigned short)((__float_as_uint(x) >> 16 & 0x8000u) | (std::is_same<T, __half>::value ? 0x3c00u : 0x3f80u));
        else if (value() == x && (bits & 0x7fffu))
            --bits;
        memcpy(&part[i], &bits, 2);
        if (finite) x -= value();
    }
    part[PARTS<T> - 1] = from_float<T>(x);
}

// Operands of a product as TF32 (10 bits after the point; the instruction ignores the bits behind them).  16-bit values are exact
// in it; an fp32 x is split in two, x = v + lo, both in integer additions (the conversion instruction took lora_grad's product with
// both operands split from 37 to 60 us).  A product is off by at most 2^-21.
//  - Beside another split one v and lo are rounded to nearest, up to 2^-23 |x|: lo is at most 2^-11 |x|, of either sign, so that
//    what is left out, the product of both low parts, 2^-22, averages out.  (Parts cut toward zero, 2^-10 and 2^-21, had three
//    times the plain fp32 sums' error.)  An infinity or NaN is lo beside a one of its sign: lo times the other's v is what x is
//    times the other, and the one times the other's parts is finite or the same infinity.
//  - Beside a whole one v is the next value below |x|, cut, so that lo has x's sign and is zero only where x is (up to 2^-22 |x|):
//    an infinite whole operand times each part is what it is times x.  An infinity is v beside the largest finite lo, a NaN is v.
//    (The last four values below fp32's end may round to infinity.)
template <bool SPLIT> struct Operand;
template <> struct Operand<false> {
    unsigned v;
};
template <> struct Operand<true> {
    unsigned v, lo;
};
template <typename T> constexpr bool IS_SPLIT = sizeof(T) == 4;

template <bool BOTH = true, typename T, int COUNT>  // BOTH: the other operand is split too
__device__ __forceinline__ void operands(const T (&x)[COUNT], Operand<IS_SPLIT<T>> (&o)[COUNT])
{
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        if constexpr (!IS_SPLIT<T>) {
            o[i].v = __float_as_uint(to_float(x[i]));
        } else if constexpr (BOTH) {
            const unsigned b = __float_as_uint(x[i]);
            const unsigned half = fabsf(x[i]) < 3.402e38f ? 0x1000u : 0u;  // beyond: cut, not rounded to infinity
            unsigned v = (b + half) & 0xffffe000u;
            unsigned lo = __float_as_uint(x[i] - __uint_as_float(v)) + half;
            if (!(fabsf(x[i]) <= FLT_MAX)) {
                v = (b & 0x80000000u) | 0x3f800000u;
                lo = __float_as_uint(x[i] + x[i]);  // a NaN's payload may lie in the bits that are ignored
            }
            o[i].v = v;
            o[i].lo = lo;
        } else {
            o[i].v = __float_as_uint(x[i] * 0.99999994f) & 0xffffe000u;  // times 1 - 2^-24: the next of fp32 below |x|
            const float left = fminf(fabsf(x[i] - __uint_as_float(o[i].v)), FLT_MAX);  // infinity - infinity becomes finite
            o[i].lo = ((__float_as_uint(x[i]) & 0x80000000u) | __float_as_uint(left)) + 0x1000u;
        }
    }
}

template <bool SA>
__device__ __forceinline__ void mma8_any(float (&d)[4], const Operand<SA> (&a)[4], const Operand<true> (&b)[2])
{
    const unsigned hi[4] = {a[0].v, a[1].v, a[2].v, a[3].v};
    if constexpr (SA) {
        const unsigned lo[4] = {a[0].lo, a[1].lo, a[2].lo, a[3].lo};
        mma8(d, lo, b[0].v, b[1].v);
    }
    mma8(d, hi, b[0].lo, b[1].lo);
    mma8(d, hi, b[0].v, b[1].v);
}

template <typename T>
__device__ __forceinline__ void store_four(T *p, const float (&y)[4])
{
    if constexpr (sizeof(T) == 4) {
        *(float4 *)p = make_float4(y[0], y[1], y[2], y[3]);
    } else {
        T u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = from_float<T>(y[e]);
        uint2 bits;
        memcpy(&bits, u, sizeof bits);
        *(uint2 *)p = bits;
    }
}

// A tile of ROWS x COLS elements whose rows are not 16-byte aligned, of which `rows` x `cols` exist (the rest: zeros), by
// COUNT threads: 4-byte asynchronous copies where rows start on 4 bytes (`words`; always in fp32), else element by element, BATCH
// loads in flight a thread (as many as leave the kernel's registers alone).
template <typename T, int ROWS, int COLS, int PITCH, int COUNT, int BATCH>
__device__ __forceinline__ void copy_loose(unsigned char *to, const T *from, long long ld, int rows, int cols, bool words, int thread)
{
    constexpr int PER = 4 / (int)sizeof(T);  // elements of a word
    static_assert(ROWS * COLS % (COUNT * PER) == 0, "whole rounds of the threads");
    if (words) {
        constexpr int ROUNDS = ROWS * COLS / PER / COUNT;
#pragma unroll BATCH
        for (int k = 0; k < ROUNDS; ++k) {
            const int at = (thread + k * COUNT) * PER, r = at / COLS, c = at % COLS;
            const int left = r < rows ? cols - c : 0, valid = left <= 0 ? 0 : left >= PER ? 4 : (int)sizeof(T);
            copy4(to + r * PITCH + c * (int)sizeof(T), valid ? from + r * ld + c : from, valid);
        }
    } else if constexpr (sizeof(T) == 2) {
        constexpr int ROUNDS = ROWS * COLS / COUNT;
        static_assert(ROUNDS % BATCH == 0, "whole batches");
#pragma unroll 1
        for (int k0 = 0; k0 < ROUNDS; k0 += BATCH) {
            unsigned short v[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const int at = thread + (k0 + k) * COUNT, r = at / COLS, c = at % COLS;
                v[k] = r < rows && c < cols ? __ldg((const unsigned short *)from + r * ld + c) : (unsigned short)0;
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const int at = thread + (k0 + k) * COUNT;
                *(unsigned short *)(to + at / COLS * PITCH + at % COLS * 2) = v[k];
            }
        }
    }
}

// ------------------------------------------------------------------ S = scale F1 In
//
// A cluster of up to 8 blocks takes TN columns, each block a part of In's rows: its 8 warps take 16 rows (8 in fp32) in turn,
// each through a ring of its own in shared memory (In's rows and F1's slice by asynchronous copies, no barrier in the loop),
// with all R x TN sums in the warp's registers.  The sums are joined over warps, then over blocks through distributed shared
// memory, in a fixed order.  With several adapters among a tile's columns the product runs once for each, and a column keeps
// its own adapter's.  It does R products for each element of In, so the tensor cores' legacy form (mma.sync, 8 cycles an
// instruction for each quarter of an SM, measured; at 1.9 GHz 576 TFLOP/s in 16 bits, 288 in TF32) is enough: In's bytes take
// as long as the products of rank 90 in 16 bits.  Measured: K 1024, 8192 columns, rank 64, bf16 (17 MB of In): 16.6 us where
// every tile has one adapter, 24.3 us where some have two, which take twice as long as the others.  Of a warp's 14200 cycles for
// its 8 steps 5300 are fragments and products, 3200 the issue of copies, 100 waits between steps and the rest the first fill;
// joining the sums takes another 7000.
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;

// Of a tile's columns: their adapters (-1: none, or past the end), and those that occur, by their first columns; for each of
// those, where there are several, which blocks of 8 columns hold any of its columns.
template <int TN>
struct TileColumns {
    __align__(16) int ids[TN];
    int list[TN], count;
    unsigned char some[TN];  // TN / 8 bits
    // `meanwhile` runs while the indices are on their way.
    template <typename F>
    __device__ __forceinline__ void load(const Columns &c, long long t0, long long N, F &&meanwhile)
    {
        const long long mine = t0 + threadIdx.x;
        const int id = threadIdx.x < TN && mine < N ? c.of(mine) : -1;
        meanwhile();
        if (threadIdx.x < TN) ids[threadIdx.x] = id;
        __syncthreads();
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            int n = 0;
            for (int b = 0; b < TN; b += 32) {
                const int t = b + lane;
                bool first = t < TN && ids[t] >= 0 && (t == 0 || ids[t] != ids[t - 1]);
                for (int s = 0; first && s < t; ++s) first = ids[s] != ids[t];
                const unsigned m = __ballot_sync(~0u, first);
                if (first) list[n + __popc(m & ((1u << lane) - 1))] = ids[t];
                n += __popc(m);
            }
            if (lane == 0) count = n;
        }
        __syncthreads();
        if (count > 1) {
            for (int d = threadIdx.x; d < count; d += THREADS) {
                const int a = list[d];
                unsigned has = 0u;
                for (int t = 0; t < TN; ++t) has |= (unsigned)(ids[t] == a) << (t >> 3);
                some[d] = (unsigned char)has;
            }
            __syncthreads();
        }
    }
};

template <typename TF, typename TI, int RT, int TN, bool TRANS>
struct ShrinkShape {
    static constexpr bool M16 = sizeof(TF) == 2 && sizeof(TI) == 2;  // 16-bit matrix instructions (else TF32)
    static constexpr int KS = sizeof(TF) == 4 ? 8 : 16;  // rows of In a step
    static constexpr int RP = RT * 16;
    // Row pitches in bytes, padded so that a matrix fragment's rows fall into different banks (ranks above 128, whose ring
    // would not fit, go without).
    static constexpr int IN_PITCH = TN * (int)sizeof(TI) + (sizeof(TI) == 4 ? 32 : 16);
    static constexpr int F_ROWS = TRANS ? KS : RP;
    static constexpr int F_COLS = TRANS ? RP : KS;
    static constexpr int F_PITCH = F_COLS * (int)sizeof(TF) + (!TRANS && RT > 8 ? 0 : TRANS && sizeof(TF) == 4 ? 32 : 16);
    static constexpr int STAGE = KS * IN_PITCH + F_ROWS * F_PITCH;
    static constexpr int S_PITCH = TN + 8;  // floats
    static constexpr int S_BYTES = RP * S_PITCH * 4;
    // Two blocks an SM where a thread's sums leave the registers for it, else one with a deeper ring.
    static constexpr int BLOCKS = RT * TN <= 128 ? 2 : 1;
    static constexpr int BUDGET = (BLOCKS == 2 ? 110 : 222) * 1024;
    static constexpr int FIT = BUDGET / (WARPS * STAGE);
    static constexpr int STAGES = FIT >= 5 ? 5 : FIT;
    static_assert(STAGES >= 2, "the ring does not fit");
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int BYTES = RING > 4 * S_BYTES ? RING : 4 * S_BYTES;  // the ring, then four warps' sums
};

template <typename TF, typename TI, int RT, int TN, bool TRANS>
__global__ void __launch_bounds__(THREADS, RT * TN <= 128 ? 2 : 1) lora_shrink(const ApplyParams p)
{
    using Q = ShrinkShape<TF, TI, RT, TN, TRANS>;
    constexpr int NB = TN / 8, RP = Q::RP, KS = Q::KS;
    constexpr bool HALF = std::is_same<TF, __half>::value;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ TileColumns<TN> tile;
    __shared__ int colmax[TN];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2;
    const long long t0 = (long long)(blockIdx.x / ranks) * TN;
    cudaTriggerProgrammaticLaunchCompletion();  // the next kernel may start: it waits for this one before it reads S
    if (threadIdx.x < TN) colmax[threadIdx.x] = 0;
    tile.load(p.c, t0, p.N, [] {});
    const int *const ids = tile.ids, *const list = tile.list;
    const int nd = tile.count;

    // ---- this block's rows of In
    float acc[RT][NB][4];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][b][e] = 0.0f;
    const long long i_begin = min(p.n1, rank * p.per1), i_end = min(p.n1, i_begin + p.per1);
    const int steps = (int)((i_end - i_begin + KS - 1) / KS);
    const int mine = steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;
    const int items = mine * nd;
    unsigned char *ring = smem + warp * (Q::STAGES * Q::STAGE);

    // A lane's 16-byte pieces of a step lie in rows first + k * (32 / CH) (CH pieces a row, a power of two), one column.
    constexpr int IN_PER = 16 / (int)sizeof(TI), IN_CH = TN / IN_PER;
    constexpr int F_PER = 16 / (int)sizeof(TF), F_CH = Q::F_COLS / F_PER;
    const int in_row = lane / IN_CH, in_col = lane % IN_CH * IN_PER;
    const long long in_left = p.N - t0 - in_col;
    const int in_bytes = in_left <= 0 ? 0 : in_left >= IN_PER ? 16 : (int)in_left * (int)sizeof(TI);
    const TI *const in_src = (const TI *)p.In + in_row * p.ldin + t0 + in_col;
    const bool in_whole = t0 + TN <= p.N, f_whole = p.R == RP;
    const long long f_ld = TRANS ? p.R : p.n1;

    auto fill = [&](int slot, int step, int a, bool with_in) {
        unsigned char *in = ring + slot * Q::STAGE, *f = in + KS * Q::IN_PITCH;
        const long long i0 = i_begin + (long long)(warp + step * WARPS) * KS;
        const int rows = (int)min((long long)KS, i_end - i0);
        if (!with_in) {
            // The step's rows are still in registers.
        } else if (p.vec_in) {
            const TI *src = in_src + i0 * p.ldin;
            unsigned char *to = in + in_row * Q::IN_PITCH + in_col * (int)sizeof(TI);
            constexpr int RS = 32 / IN_CH;
            if (rows == KS && in_whole) {
#pragma unroll
                for (int k = 0; k < KS * IN_CH / 32; ++k) copy16(to + k * RS * Q::IN_PITCH, src + k * RS * p.ldin, 16);
            } else {
#pragma unroll
                for (int k = 0; k < KS * IN_CH / 32; ++k) {
                    const int valid = in_row + k * RS < rows ? in_bytes : 0;
                    copy16(to + k * RS * Q::IN_PITCH, valid ? src + k * RS * p.ldin : (const TI *)p.In, valid);
                }
            }
        } else {
            copy_loose<TI, KS, TN, Q::IN_PITCH, 32, 4>(in, (const TI *)p.In + i0 * p.ldin + t0, p.ldin, rows, (int)min((long long)TN, p.N - t0), p.word_in, lane);
        }
        const TF *F = (const TF *)p.F1 + (long long)a * p.R * p.n1 + (TRANS ? i0 * p.R : i0);
        if (p.vec_f1) {
            constexpr int COUNT = Q::F_ROWS * F_CH;
            if (rows == KS && f_whole && COUNT % 32 == 0 && (F_CH <= 32 && 32 % F_CH == 0)) {
                const TF *src = F + lane / F_CH * f_ld + lane % F_CH * F_PER;
                unsigned char *to = f + lane / F_CH * Q::F_PITCH + lane % F_CH * 16;
#pragma unroll
                for (int k = 0; k < COUNT / 32; ++k) copy16(to + k * (32 / F_CH) * Q::F_PITCH, src + k * (32 / F_CH) * f_ld, 16);
            } else {
#pragma unroll
                for (int k = 0; k < (COUNT + 31) / 32; ++k) {
                    const int r = (lane + k * 32) / F_CH, c = (lane + k * 32) % F_CH * F_PER;
                    const int left = TRANS ? (r < rows ? p.R - c : 0) : (r < p.R ? rows - c : 0);
                    const int valid = left <= 0 ? 0 : left >= F_PER ? 16 : left * (int)sizeof(TF);
                    if (COUNT % 32 == 0 || lane + k * 32 < COUNT)
                        copy16(f + r * Q::F_PITCH + c * (int)sizeof(TF), valid ? F + r * f_ld + c : (const TF *)p.F1, valid);
                }
            }
        } else {
            copy_loose<TF, Q::F_ROWS, Q::F_COLS, Q::F_PITCH, 32, 4>(f, F, f_ld, TRANS ? rows : p.R, TRANS ? p.R : rows, p.word_f1, lane);
        }
    };

    {
        int next_step = 0, next_d = 0, filled = 0, slot = 0;
        auto fill_next = [&]() {
            if (filled < items) {
                fill(slot, next_step, list[next_d], !Q::M16 || next_d == 0);
                if (++next_d == nd) {
                    next_d = 0;
                    ++next_step;
                }
                ++filled;
                if (++slot == Q::STAGES) slot = 0;
            }
            copy_commit();
        };
        for (int s = 0; s < Q::STAGES - 1; ++s) fill_next();
        int d = 0, at = 0;
        unsigned B[Q::M16 ? NB : 1][2];
        for (int it = 0; it < items; ++it) {
            copy_wait<Q::STAGES - 2>();
            __syncwarp();  // the copies of all lanes have landed, and the slot filled next has been read by all
            fill_next();
            const unsigned char *in = ring + at * Q::STAGE, *f = in + KS * Q::IN_PITCH;
            if (++at == Q::STAGES) at = 0;
            const int a = list[d], this_d = d;
            const bool first = d == 0;
            if (++d == nd) d = 0;
            const unsigned some = nd > 1 ? tile.some[this_d] : ~0u;
            // acc += part; with several adapters, only in the blocks with any of adapter a's columns, and only for these.
            auto add = [&](auto &&product) {
                if (nd == 1) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int m = 0; m < RT; ++m) {
                            if constexpr (sizeof(TF) == 4) {
                                // The tensor cores cut their sums instead of rounding them: in fp32 long sums are kept outside.
                                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                product(m, b, part);
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[m][b][e] += part[e];
                            } else {
                                product(m, b, acc[m][b]);
                            }
                        }
                    return;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (!(some >> b & 1)) continue;
                    const bool own[2] = {ids[b * 8 + 2 * q] == a, ids[b * 8 + 2 * q + 1] == a};
#pragma unroll
                    for (int m = 0; m < RT; ++m) {
                        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        product(m, b, part);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (own[e & 1]) acc[m][b][e] += part[e];
                    }
                }
            };
            if constexpr (Q::M16) {
                unsigned A[RT][4];
#pragma unroll
                for (int m = 0; m < RT; ++m)
                    load_matrices<TRANS>(A[m], TRANS ? f + ((lane & 7) + (lane >> 4) * 8) * Q::F_PITCH + (m * 16 + (lane >> 3 & 1) * 8) * 2
                                                     : f + (m * 16 + (lane & 15)) * Q::F_PITCH + (lane >> 4) * 16);
                if (first) {  // the step's rows stay in registers for its other adapters
#pragma unroll
                    for (int b = 0; b < NB; b += 2) {
                        unsigned t[4];
                        load_matrices<true>(t, in + (lane & 15) * Q::IN_PITCH + (b + (lane >> 4)) * 16);
                        B[b][0] = t[0];
                        B[b][1] = t[1];
                        B[b + 1][0] = t[2];
                        B[b + 1][1] = t[3];
                    }
                }
                add([&](int m, int b, float (&to)[4]) { mma16<TF>(to, A[m], B[b][0], B[b][1]); });
            } else {
#pragma unroll
                for (int k = 0; k < KS; k += 8) {
                    Operand<IS_SPLIT<TF>> A[RT][4];
#pragma unroll
                    for (int m = 0; m < RT; ++m) {
                        TF v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = m * 16 + g + (e & 1) * 8, i = k + q + (e >> 1) * 4;
                            v[e] = *(const TF *)(TRANS ? f + i * Q::F_PITCH + r * sizeof(TF) : f + r * Q::F_PITCH + i * sizeof(TF));
                        }
                        operands(v, A[m]);
                    }
                    Operand<true> B8[2];
                    int have = -1;
                    add([&](int m, int b, float (&to)[4]) {
                        if (have != b) {
                            TI v[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) v[e] = *(const TI *)(in + (k + q + e * 4) * Q::IN_PITCH + (b * 8 + g) * sizeof(TI));
                            operands<IS_SPLIT<TF>>(v, B8);
                            have = b;
                        }
                        mma8_any(to, A[m], B8);
                    });
                }
            }
        }
        copy_wait<0>();
    }
    __syncthreads();

    // ---- S joined over the warps: 4 to 7 leave theirs, 0 to 3 add them to their own
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
    for (int i = threadIdx.x; i < RP * TN; i += THREADS) {
        float *s = slot + i / TN * PITCH + i % TN;
        s[0] = (s[0] + s[SLOT]) + (s[2 * SLOT] + s[3 * SLOT]);
    }
    auto sync_all = [&]() {
        if (ranks > 1)
            cluster.sync();
        else
            __syncthreads();
    };
    sync_all();

    // ---- S joined over the blocks: each takes TN / ranks columns (a power of two: a thread keeps one)
    const int own = TN / ranks;
    const int c = rank * own + (threadIdx.x & (own - 1)), a = ids[c];
    const int r_first = threadIdx.x / own, r_step = THREADS / own;
    const float scale = a < 0 ? 0.0f : p.scale ? __ldg(p.scale + a) : 1.0f;
    const Hidden h(p.hidden, p.R, p.N);
    const int place = Hidden::place(c);
    const bool keep = t0 + c < h.pitch;
    float most = 0.0f;
    for (int r = r_first; r < p.R; r += r_step) {
        float v = 0.0f;
        if (ranks == 1) {
            v = slot[r * PITCH + c];
        } else {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = k < ranks ? cluster.map_shared_rank(slot, k)[r * PITCH + c] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v += x[k];
        }
        v = a >= 0 ? v * scale : 0.0f;  // whatever a column without an adapter has gathered
        if (keep) h.s()[r * h.pitch + t0 + c] = v;
        if (HALF) {
            slot[SLOT + r * PITCH + c] = v;
            if (fabsf(v) <= FLT_MAX) most = fmaxf(most, fabsf(v));
        } else if (sizeof(TF) == 2 && keep) {
            TF part[PARTS<TF>];
            split16<TF>(v, part);
#pragma unroll
            for (int i = 0; i < PARTS<TF>; ++i) h.part<TF>(i)[r * h.pitch + t0 + place] = part[i];
        }
    }
    if (HALF) {
        atomicMax(&colmax[c], __float_as_int(most));  // the order does not matter
        __syncthreads();
        // The column's largest finite value goes to [2^13, 2^14), whatever stands beside it; zeros stay.
        const int e = (colmax[c] >> 23) - 127;
        const int shift = e == -127 ? 0 : max(-126, e - 13);
        const float down = __int_as_float((127 - shift) << 23);
        if (keep) {
            for (int r = r_first; r < p.R; r += r_step) {
                TF part[PARTS<TF>];
                split16<TF>(slot[SLOT + r * PITCH + c] * down, part);
#pragma unroll
                for (int i = 0; i < PARTS<TF>; ++i) h.part<TF>(i)[r * h.pitch + t0 + place] = part[i];
            }
            if (r_first == 0) h.colscale()[t0 + c] = __int_as_float((127 + shift) << 23);
        }
    }
    if (ranks > 1) cluster.sync();  // the others have read this block's sums
}

// ------------------------------------------------------------------ Out = base + F2 S
//
// A block takes 64 columns and up to 8 chunks of 128 rows of Out, a warp 16 rows of a chunk.  S's columns stay in shared
// memory; F2's slices come a chunk ahead and base two (asynchronous copies), the first of them before the block waits for the
// kernel that makes S (programmatic dependent launch), so that the start of this kernel hides behind the end of that
// one.  Columns are dealt to the matrix instruction so that a thread's results of two blocks of 8 lie side by side: base and
// Out move 16 bytes a thread.  In 16 bits S's parts are multiplied one by one, so that Out is, before its own rounding,
// as exact as fp32 sums of exact products.  With several adapters among the columns the product runs once for each, for the
// pairs of blocks that have any of its columns.  Bound by base and Out: R / 8 products a byte.
// Measured: M 4096, 8192 columns, rank 64, bf16 factors, fp32 base and Out (268 MB), three parts of S, at 1, 2, 3, 4, 5, 8 and
// 16 chunks a block: 96, 77, 73, 70, 72, 72, 70 us (3.7 TB/s at 3) where every tile has one adapter, 97, 85, 81, 82, 86, 91,
// 108 us where some have two, whose blocks end last.  Two parts of S took 6 us less.
constexpr int EXP_COLS = 64;
constexpr int EXP_ROWS = WARPS * 16;
constexpr int EXP_PAIRS = EXP_COLS / 16;

template <typename TF, int RT, bool TRANS>
struct ExpandShape {
    static constexpr int COUNT = sizeof(TF) == 2 ? PARTS<TF> : 1;  // S's parts
    static constexpr int RP = RT * 16;
    static constexpr int F_ROWS = TRANS ? RP : 16;
    static constexpr int F_COLS = TRANS ? 16 : RP;
    static constexpr int F_PITCH = F_COLS * (int)sizeof(TF) + (!TRANS || sizeof(TF) == 2 ? 16 : RT > 8 ? 0 : 32);
    static constexpr int F_BYTES = F_ROWS * F_PITCH;
    static constexpr int S_PITCH = EXP_COLS * (int)sizeof(TF) + (sizeof(TF) == 4 ? 32 : 16);
    static constexpr int S_BYTES = RP * S_PITCH;  // one part
    static constexpr int S_ALL = S_BYTES * COUNT;
    // Two blocks an SM up to rank 64, else one; two chunks of base ahead, or as many as fit; F2's slices in two buffers where
    // they fit.
    static constexpr int BLOCKS = RT <= 4 ? 2 : 1;
    static constexpr int ROOM = BLOCKS == 2 ? 112 * 1024 : 222 * 1024;
    static constexpr int SLOT = EXP_PAIRS * 2 * 16 * THREADS;
    static constexpr int LEAST = S_ALL + WARPS * F_BYTES;
    static constexpr int SLOTS = LEAST + 2 * SLOT <= ROOM ? 2 : LEAST + SLOT <= ROOM ? 1 : 0;
    static constexpr int BUFFERS = LEAST + SLOTS * SLOT + WARPS * F_BYTES <= ROOM ? 2 : 1;
    static constexpr int BYTES = S_ALL + SLOTS * SLOT + BUFFERS * WARPS * F_BYTES;
    static_assert(BYTES <= ROOM, "F2's slices do not fit");
};

template <typename TF, int RT, bool TRANS>
__global__ void __launch_bounds__(THREADS, RT <= 4 ? 2 : 1) lora_expand(const ApplyParams p)
{
    using Q = ExpandShape<TF, RT, TRANS>;
    constexpr int COUNT = Q::COUNT;
    constexpr bool HALF = std::is_same<TF, __half>::value;
    constexpr int PAIRS = EXP_PAIRS, RP = Q::RP;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ TileColumns<EXP_COLS> tile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2;
    const unsigned across = (unsigned)((p.N + EXP_COLS - 1) / EXP_COLS);  // neighbouring blocks share rows
    const long long t0 = (long long)(blockIdx.x % across) * EXP_COLS;
    const long long j_first = (long long)(blockIdx.x / across) * p.chunks * EXP_ROWS + warp * 16;
    const int chunks = (int)max(0ll, min((long long)p.chunks, (p.n2 - j_first + EXP_ROWS - 1) / EXP_ROWS));  // this warp's
    const int last_rows = chunks > 0 ? (int)min(16ll, p.n2 - j_first - (long long)(chunks - 1) * EXP_ROWS) : 0;
    unsigned char *const sh = smem, *const f0 = smem + Q::S_ALL + warp * (Q::BUFFERS * Q::F_BYTES);
    unsigned char *const slots = smem + Q::S_ALL + WARPS * Q::BUFFERS * Q::F_BYTES + threadIdx.x * 16;  // pieces THREADS * 16 apart
    __shared__ __align__(16) float colscale[EXP_COLS];

    const int base_size = p.basetype == 0 ? 4 : 2;
    const unsigned char *base = (const unsigned char *)p.base + ((j_first + g) * p.ldbase + t0 + 4 * q) * base_size;
    const bool fetch = Q::SLOTS > 0 && p.base && t0 + EXP_COLS <= p.N && p.vec_base;  // base comes by asynchronous copies
    const long long base_step = (long long)EXP_ROWS * p.ldbase * base_size, base_down = 8 * p.ldbase * base_size;
    auto fetch_base = [&](int chunk, const unsigned char *at, int rows) {  // a chunk's part of base, into its slot
        unsigned char *const slot = slots + (Q::SLOTS == 2 ? (chunk & 1) * Q::SLOT : 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int valid = g + h * 8 < rows ? 16 : 0;
            const unsigned char *row = valid ? at + (h ? base_down : 0) : (const unsigned char *)p.base;
#pragma unroll
            for (int b = 0; b < PAIRS; ++b) {
                if (base_size == 4)
                    copy16(slot + (b * 2 + h) * (THREADS * 16), row + (valid ? b * 64 : 0), valid);
                else
                    copy8(slot + (b * 2 + h) * (THREADS * 16), row + (valid ? b * 32 : 0), valid >> 1);
            }
        }
    };
    const long long f_ld = TRANS ? p.n2 : p.R;
    auto fill_f = [&](unsigned char *f, int a, int chunk, int rows) {  // the warp's rows of adapter a's F2
        const long long j0 = j_first + (long long)chunk * EXP_ROWS;
        const TF *F = (const TF *)p.F2 + (long long)a * p.R * p.n2 + (TRANS ? j0 : j0 * p.R);
        constexpr int PER = 16 / (int)sizeof(TF), CH = Q::F_COLS / PER, PIECES = Q::F_ROWS * CH;
        if (p.vec_f2) {
#pragma unroll
            for (int k = 0; k < (PIECES + 31) / 32; ++k) {
                const int r = (lane + k * 32) / CH, c = (lane + k * 32) % CH * PER;
                const int left = TRANS ? (r < p.R ? rows - c : 0) : (r < rows ? p.R - c : 0);
                const int valid = left <= 0 ? 0 : left >= PER ? 16 : left * (int)sizeof(TF);
                if (PIECES % 32 == 0 || lane + k * 32 < PIECES)
                    copy16(f + r * Q::F_PITCH + c * (int)sizeof(TF), valid ? F + r * f_ld + c : (const TF *)p.F2, valid);
            }
        } else {
            copy_loose<TF, Q::F_ROWS, Q::F_COLS, Q::F_PITCH, 32, 2>(f, F, f_ld, TRANS ? p.R : rows, TRANS ? rows : p.R, p.word_f2, lane);
        }
    };
    auto rows_of = [&](int chunk) { return chunk >= chunks ? 0 : chunk == chunks - 1 ? last_rows : 16; };

    const Hidden hid(p.hidden, p.R, p.N);
    tile.load(p.c, t0, p.N, [&] {  // while the indices are on their way: base, and S's columns
        if (fetch) {
            fetch_base(0, base, rows_of(0));
            if (Q::SLOTS == 2 && chunks > 1) fetch_base(1, base + base_step, rows_of(1));
        }
        cudaGridDependencySynchronize();
        cudaTriggerProgrammaticLaunchCompletion();
        constexpr int PER = 16 / (int)sizeof(TF), CH = EXP_COLS / PER;
        const int c = threadIdx.x % CH * PER, r = threadIdx.x / CH;
#pragma unroll
        for (int part = 0; part < COUNT; ++part) {
            const TF *const src = sizeof(TF) == 4 ? (const TF *)hid.s() : hid.template part<TF>(part);
#pragma unroll
            for (int k = 0; k < (RP * CH + THREADS - 1) / THREADS; ++k) {
                const int row = r + k * (THREADS / CH), valid = row < p.R ? 16 : 0;
                if (RP * CH % THREADS == 0 || row < RP)
                    copy16(sh + part * Q::S_BYTES + row * Q::S_PITCH + c * (int)sizeof(TF), valid ? src + row * hid.pitch + t0 + c : src, valid);
            }
        }
        if (HALF && threadIdx.x < EXP_COLS) colscale[threadIdx.x] = hid.colscale()[t0 + threadIdx.x];
    });
    const int *const ids = tile.ids, *const list = tile.list;
    const int nd = tile.count;
    if (nd > 0 && chunks > 0) fill_f(f0, list[0], 0, rows_of(0));
    // A bit for each of a thread's columns (4 q + (k & 3) of pair k / 4): it exists, has an adapter.
    unsigned exist = 0u, has = 0u;
#pragma unroll
    for (int b = 0; b < PAIRS; ++b) {
        const int4 id = *(const int4 *)(ids + b * 16 + 4 * q);
        has |= ((id.x >= 0) | (id.y >= 0) << 1 | (id.z >= 0) << 2 | (id.w >= 0) << 3) << (b * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) exist |= (unsigned)(t0 + b * 16 + 4 * q + e < p.N) << (b * 4 + e);
    }
    // The usual tile, without masks: one adapter for all of its columns, everything aligned.
    const bool plain = __all_sync(~0u, has == 0xffffu) && nd == 1 && p.vec_out && p.vec_f2 && (fetch || !p.base);
    copy_commit();
    copy_wait<0>();
    __syncthreads();

    float sum[PAIRS][2][4];  // [pair][block of the pair][e]: rows g, g + 8; columns 16 pair + 4 q + 2 block + (e & 1)
    auto multiply = [&](const unsigned char *f, auto all, unsigned some) {  // all: every pair, whatever `some` says
#pragma unroll
        for (int b = 0; b < PAIRS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[b][h][e] = 0.0f;
        if constexpr (sizeof(TF) == 2) {
#pragma unroll(RT <= 4 ? RT : 2)
            for (int k = 0; k < RT; ++k) {
                unsigned A[4];
                load_matrices<TRANS>(A, TRANS ? f + (k * 16 + (lane & 7) + (lane >> 4) * 8) * Q::F_PITCH + (lane >> 3 & 1) * 16
                                              : f + (lane & 15) * Q::F_PITCH + (k * 16 + (lane >> 4) * 8) * 2);
                const int row = (k * 16 + (lane & 15)) * Q::S_PITCH + (lane >> 4) * 16;
#pragma unroll
                for (int b = 0; b < PAIRS; ++b) {
                    if (!all.value && !(some >> b & 1)) continue;
#pragma unroll
                    for (int part = COUNT - 1; part >= 0; --part) {
                        unsigned B[4];
                        load_matrices<true>(B, sh + part * Q::S_BYTES + row + b * 32);
                        mma16<TF>(sum[b][0], A, B[0], B[1]);
                        mma16<TF>(sum[b][1], A, B[2], B[3]);
                    }
                }
            }
        } else {
#pragma unroll 2
            for (int k = 0; k < RP; k += 8) {
                Operand<true> A[4];
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = g + (e & 1) * 8, r = k + q + (e >> 1) * 4;
                    v[e] = *(const float *)(TRANS ? f + r * Q::F_PITCH + j * 4 : f + j * Q::F_PITCH + r * 4);
                }
                operands(v, A);
#pragma unroll
                for (int b = 0; b < PAIRS; ++b) {
                    if (!all.value && !(some >> b & 1)) continue;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const unsigned char *s = sh + (k + q) * Q::S_PITCH + (b * 16 + 4 * (g >> 1) + 2 * h + (g & 1)) * 4;
                        const float w[2] = {*(const float *)s, *(const float *)(s + 4 * Q::S_PITCH)};
                        Operand<true> B[2];
                        operands(w, B);
                        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // the tensor cores cut their sums: kept outside
                        mma8_any(part, A, B);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[b][h][e] += part[e];
                    }
                }
            }
        }
    };
    const int out_size = p.outtype == 0 ? 4 : 2;
    unsigned char *out = (unsigned char *)p.Out + ((j_first + g) * p.ldout + t0 + 4 * q) * out_size;
    auto store = [&](auto type, const float (&y)[PAIRS][2][4], int rows) {
        using TO = std::conditional_t<type.value == 0, float, std::conditional_t<type.value == 1, __half, __nv_bfloat16>>;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (g + h * 8 >= rows) continue;
            TO *row = (TO *)out + h * 8 * p.ldout;
#pragma unroll
            for (int b = 0; b < PAIRS; ++b) {
                const unsigned w = exist >> (b * 4) & 15u;
                if (p.vec_out && w == 15u) {
                    store_four(row + b * 16, y[b][h]);
                } else if (w) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (w >> e & 1) row[b * 16 + e] = from_float<TO>(y[b][h][e]);
                }
            }
        }
    };

    const long long out_step = (long long)EXP_ROWS * p.ldout * out_size;
    int chunk = 0;
    if (plain) {
        // Whole chunks of a usual tile: a lane's pieces of F2's slice lie CH pieces apart in one column (or row), all
        // addresses advance by constants, and the next chunk's copies are under way while this one is multiplied.
        constexpr int PER = 16 / (int)sizeof(TF), CH = Q::F_COLS / PER, PIECES = Q::F_ROWS * CH;
        constexpr int ROWS = CH >= 32 ? 1 : 32 / CH;  // rows from a lane's piece to its next
        const int f_row = lane / CH, f_col = lane % CH * PER;
        const TF *f_src = (const TF *)p.F2 + (long long)list[0] * p.R * p.n2 + (TRANS ? j_first : j_first * p.R) + f_row * f_ld + f_col;
        const long long f_step = TRANS ? EXP_ROWS : (long long)EXP_ROWS * p.R;
        const bool simple = CH <= 32 && PIECES % 32 == 0 && (TRANS ? true : f_col + PER <= p.R || f_col >= p.R);
        auto fetch_f = [&](unsigned char *f, const TF *src) {
            unsigned char *to = f + f_row * Q::F_PITCH + f_col * (int)sizeof(TF);
#pragma unroll
            for (int k = 0; k < PIECES / 32; ++k) {
                const bool in = TRANS ? f_row + k * ROWS < p.R : f_col < p.R;
                copy16(to + k * ROWS * Q::F_PITCH, in ? src + k * ROWS * f_ld : (const TF *)p.F2, in ? 16 : 0);
            }
        };
        auto run = [&](auto base_type, auto out_type) {  // base_type -1: none
            using TO = std::conditional_t<out_type.value == 0, float, std::conditional_t<out_type.value == 1, __half, __nv_bfloat16>>;
            constexpr bool B32 = base_type.value == 0, B16 = base_type.value > 0;
            // F2's slice of the next chunk, then base of the one after it: in groups of their own, so that the wait for the
            // first leaves the second under way.
            auto fetch_next = [&]() {
                if (chunk + 1 < chunks) {
                    f_src += f_step;
                    unsigned char *const f = f0 + (Q::BUFFERS == 2 ? (chunk + 1 & 1) * Q::F_BYTES : 0);
                    if (rows_of(chunk + 1) == 16 && simple)
                        fetch_f(f, f_src);
                    else
                        fill_f(f, list[0], chunk + 1, rows_of(chunk + 1));
                }
                copy_commit();
                if ((B32 || B16) && chunk + Q::SLOTS < chunks) {
                    const unsigned char *at = base + Q::SLOTS * base_step;
                    if (rows_of(chunk + Q::SLOTS) == 16) {
                        unsigned char *const slot = slots + (Q::SLOTS == 2 ? (chunk & 1) * Q::SLOT : 0);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int b = 0; b < PAIRS; ++b) {
                                const unsigned char *src = at + (h ? base_down : 0) + b * (B32 ? 64 : 32);
                                if (B32)
                                    copy16(slot + (b * 2 + h) * (THREADS * 16), src, 16);
                                else
                                    copy8(slot + (b * 2 + h) * (THREADS * 16), src, 8);
                            }
                    } else {
                        fetch_base(chunk + Q::SLOTS, at, rows_of(chunk + Q::SLOTS));
                    }
                }
                copy_commit();
            };
            for (; chunk < chunks && rows_of(chunk) == 16; ++chunk, out += out_step, base += base_step) {
                copy_wait<Q::SLOTS == 2 ? 1 : 0>();
                __syncwarp();
                const unsigned char *const slot = slots + (Q::SLOTS == 2 ? (chunk & 1) * Q::SLOT : 0);
                float4 old[B32 ? PAIRS * 2 : 1];
                uint2 old16[B16 ? PAIRS * 2 : 1];
                if (B32) {
#pragma unroll
                    for (int i = 0; i < PAIRS * 2; ++i) old[i] = *(const float4 *)(slot + i * (THREADS * 16));
                }
                if (B16) {
#pragma unroll
                    for (int i = 0; i < PAIRS * 2; ++i) old16[i] = *(const uint2 *)(slot + i * (THREADS * 16));
                }
                if (Q::BUFFERS == 2) fetch_next();
                multiply(f0 + (Q::BUFFERS == 2 ? (chunk & 1) * Q::F_BYTES : 0), std::true_type{}, 0u);
                if (Q::BUFFERS == 1) {
                    __syncwarp();
                    fetch_next();
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    TO *row = (TO *)out + h * 8 * p.ldout;
#pragma unroll
                    for (int b = 0; b < PAIRS; ++b) {
                        float y[4] = {sum[b][0][2 * h], sum[b][0][2 * h + 1], sum[b][1][2 * h], sum[b][1][2 * h + 1]};
                        if (HALF) {
                            const float4 c = *(const float4 *)(colscale + b * 16 + 4 * q);
                            y[0] *= c.x;
                            y[1] *= c.y;
                            y[2] *= c.z;
                            y[3] *= c.w;
                        }
                        if (B32) {
                            y[0] += old[b * 2 + h].x;
                            y[1] += old[b * 2 + h].y;
                            y[2] += old[b * 2 + h].z;
                            y[3] += old[b * 2 + h].w;
                        }
                        if (B16) {
                            y[0] += as_float(old16[b * 2 + h].x & 0xffffu, base_type.value);
                            y[1] += as_float(old16[b * 2 + h].x >> 16, base_type.value);
                            y[2] += as_float(old16[b * 2 + h].y & 0xffffu, base_type.value);
                            y[3] += as_float(old16[b * 2 + h].y >> 16, base_type.value);
                        }
                        store_four(row + b * 16, y);
                    }
                }
            }
        };
        // base has Out's type, or is fp32 beside a 16-bit Out, or there is none.
        const auto with_base = [&](auto out_type) {
            if (!p.base)
                run(std::integral_constant<int, -1>{}, out_type);
            else if (p.basetype == 0)
                run(std::integral_constant<int, 0>{}, out_type);
            else
                run(out_type, out_type);
        };
        if (p.outtype == 0)
            with_base(std::integral_constant<int, 0>{});
        else if (p.outtype == 1)
            with_base(std::integral_constant<int, 1>{});
        else
            with_base(std::integral_constant<int, 2>{});
    }
    for (int turn = chunk; chunk < chunks; ++chunk, out += out_step, base += base_step) {
        const int rows = rows_of(chunk);
        copy_wait<0>();
        __syncwarp();
        float old[PAIRS][2][4];  // rows g, g + 8; columns 16 pair + 4 q ...
#pragma unroll
        for (int b = 0; b < PAIRS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const unsigned char *at = slots + (Q::SLOTS == 2 ? (chunk & 1) * Q::SLOT : 0) + (b * 2 + h) * (THREADS * 16);
                if (fetch && base_size == 4) {
                    v = *(const float4 *)at;
                } else if (fetch) {
                    const uint2 u = *(const uint2 *)at;
                    v = make_float4(as_float(u.x & 0xffffu, p.basetype), as_float(u.x >> 16, p.basetype), as_float(u.y & 0xffffu, p.basetype),
                                    as_float(u.y >> 16, p.basetype));
                } else if (p.base && g + h * 8 < rows) {
                    const unsigned char *from = base + (h ? base_down : 0);
                    const auto element = [&](int e) {
                        return t0 + b * 16 + 4 * q + e >= p.N ? 0.0f
                               : base_size == 4               ? ((const float *)from)[b * 16 + e]
                                                              : as_float(((const unsigned short *)from)[b * 16 + e], p.basetype);
                    };
                    v = make_float4(element(0), element(1), element(2), element(3));
                }
                old[b][h][0] = v.x;
                old[b][h][1] = v.y;
                old[b][h][2] = v.z;
                old[b][h][3] = v.w;
            }
        if (chunk + Q::SLOTS < chunks && fetch) fetch_base(chunk + Q::SLOTS, base + Q::SLOTS * base_step, rows_of(chunk + Q::SLOTS));
        copy_commit();
        for (int pass = 0; pass < nd; ++pass) {
            // The thread's columns of this pass's adapter; pairs of blocks with any.
            const int a = list[pass];
            const unsigned blocks = nd > 1 ? tile.some[pass] : ~0u;
            unsigned mine = 0u, some = 0u;
#pragma unroll
            for (int b = 0; b < PAIRS; ++b) {
                const int4 id = *(const int4 *)(ids + b * 16 + 4 * q);
                mine |= ((id.x == a) | (id.y == a) << 1 | (id.z == a) << 2 | (id.w == a) << 3) << (b * 4);
                some |= (unsigned)((blocks >> (2 * b) & 3u) != 0u) << b;
            }
            // F2's slices alternate between two buffers: the next pass's (or chunk's) is fetched during this one.
            const bool more = pass + 1 < nd || chunk + 1 < chunks;
            const int next_pass = pass + 1 < nd ? pass + 1 : 0, next_chunk = pass + 1 < nd ? chunk : chunk + 1;
            if (pass > 0) {
                copy_wait<0>();
                __syncwarp();
            }
            if (Q::BUFFERS == 2 && more) fill_f(f0 + (turn + 1 & 1) * Q::F_BYTES, list[next_pass], next_chunk, rows_of(next_chunk));
            copy_commit();
            multiply(Q::BUFFERS == 2 ? f0 + (turn & 1) * Q::F_BYTES : f0, std::false_type{}, some);
            __syncwarp();
            if (Q::BUFFERS == 1 && more) fill_f(f0, list[next_pass], next_chunk, rows_of(next_chunk));
            copy_commit();
            ++turn;
#pragma unroll
            for (int b = 0; b < PAIRS; ++b) {
                float4 c = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                if (HALF) c = *(const float4 *)(colscale + b * 16 + 4 * q);
                const float by[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (mine >> (b * 4 + e) & 1) old[b][h][e] += sum[b][e >> 1][2 * h + (e & 1)] * by[e];
            }
        }
        if (p.outtype == 0)
            store(std::integral_constant<int, 0>{}, old, rows);
        else if (p.outtype == 1)
            store(std::integral_constant<int, 1>{}, old, rows);
        else
            store(std::integral_constant<int, 2>{}, old, rows);
    }
}

// ------------------------------------------------------------------ few columns
//
// A cluster of 8 blocks for one column, where a matrix instruction's 8 columns would mostly stand empty: each block takes an
// eighth of D's columns (a lane 16 bytes of a row), the blocks add their R sums through distributed shared memory, and each
// takes an eighth of U's rows, whose first loads start before the sums are joined.  fp32 sums throughout.  A call is bound
// by its latency, many columns by the reads of their factors from L2.  Measured (fp16, 64 adapters of rank 16, 4096 x 1024):
// 1 column 5.1 us, 32 columns 6.4 us, 64 columns 9 us, where the tiles take 10, 61 and 61 us.
constexpr int TOKEN_RANKS = 8;

// Element i of base (which may be Out: no read-only loads).
__device__ __forceinline__ float load_base(const ApplyParams &p, long long i)
{
    return p.basetype == 0 ? ((const float *)p.base)[i] : as_float(((const unsigned short *)p.base)[i], p.basetype);
}

template <typename T, int VEC1, int VEC2>
__global__ void __launch_bounds__(THREADS, 4) lora_token(const ApplyParams p)
{
    constexpr int AHEAD = 4;  // rows of U in flight a thread
    extern __shared__ __align__(16) float xs[];  // the block's part of the column
    __shared__ float part[256], H[256 + 8];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long t = blockIdx.x / TOKEN_RANKS;
    const int a = p.c.of(t);
    const long long per2 = (p.n2 + TOKEN_RANKS - 1) / TOKEN_RANKS;
    const long long m0 = min(p.n2, rank * per2), m1 = min(p.n2, m0 + per2);
    if (a < 0) {  // the same in all blocks of the cluster
        for (long long m = m0 + threadIdx.x; m < m1; m += THREADS)
            store_as(p.Out, p.outtype, m * p.ldout + t, p.base ? load_base(p, m * p.ldbase + t) : 0.0f);
        return;
    }
    // U: lanes2 threads a row; their rows' first loads.
    const T *const U = (const T *)p.F2 + (long long)a * p.R * p.n2;
    const int pieces2 = (p.R + VEC2 - 1) / VEC2;
    int lanes2 = 1;
    while (lanes2 < 32 && lanes2 < pieces2) lanes2 *= 2;
    const int l2 = threadIdx.x & (lanes2 - 1), per_pass = THREADS / lanes2;
    long long m = m0 + threadIdx.x / lanes2;
    Pack<T, VEC2> u[AHEAD];
    float old[AHEAD];
    auto load_u = [&](long long first) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const long long row = first + (long long)k * per_pass;
            u[k].zero();
            old[k] = 0.0f;
            if (row < m1) {
                if (l2 < pieces2) u[k].load(U + row * p.R + l2 * VEC2);
                if (l2 == 0 && p.base) old[k] = load_base(p, row * p.ldbase + t);
            }
        }
    };
    load_u(m);

    const long long k0 = min(p.n1, rank * p.per1), len = min(p.n1, k0 + p.per1) - k0;
    for (long long i = threadIdx.x; i < len; i += THREADS) xs[i] = to_float(((const T *)p.In)[(k0 + i) * p.ldin + t]);
    for (int r = p.R + (int)threadIdx.x; r < 256 + 8; r += THREADS) H[r] = 0.0f;
    __syncthreads();
    // D: lanes1 threads a row.
    const T *const D = (const T *)p.F1 + (long long)a * p.R * p.n1 + k0;
    int lanes1 = 1;
    while (lanes1 < 32 && lanes1 * VEC1 < len) lanes1 *= 2;
    const int l1 = lane & (lanes1 - 1), sub = lane / lanes1, rows1 = 32 / lanes1;
#pragma unroll 4
    for (int r0 = warp * rows1; r0 < p.R; r0 += WARPS * rows1) {
        const int r = r0 + sub;
        float v = 0.0f;
        if (r < p.R) {
#pragma unroll 2
            for (long long i = l1 * VEC1; i < len; i += lanes1 * VEC1) {
                Pack<T, VEC1> d;
                d.load(D + r * p.n1 + i);
#pragma unroll
                for (int e = 0; e < VEC1; ++e) v += d.get(e) * xs[i + e];
            }
        }
        for (int o = lanes1 >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        if (l1 == 0 && r < p.R) part[r] = v;
    }
    cluster.sync();
    if (threadIdx.x < p.R) {
        float x[TOKEN_RANKS], v = 0.0f;
#pragma unroll
        for (int k = 0; k < TOKEN_RANKS; ++k) x[k] = cluster.map_shared_rank(part, k)[threadIdx.x];
#pragma unroll
        for (int k = 0; k < TOKEN_RANKS; ++k) v += x[k];
        H[threadIdx.x] = p.scale ? v * __ldg(p.scale + a) : v;
    }
    cluster.barrier_arrive();
    __syncthreads();
    for (; m - (int)threadIdx.x / lanes2 < m1; m += (long long)AHEAD * per_pass) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const long long row = m + (long long)k * per_pass;
            float v = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC2; ++e) v += u[k].get(e) * H[min(l2, pieces2 - 1) * VEC2 + e];
            if (l2 >= pieces2) v = 0.0f;
            for (int c = l2 + lanes2; c < pieces2 && row < m1; c += lanes2) {
                Pack<T, VEC2> w;
                w.load(U + row * p.R + c * VEC2);
#pragma unroll
                for (int e = 0; e < VEC2; ++e) v += w.get(e) * H[c * VEC2 + e];
            }
            for (int o = lanes2 >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
            if (l2 == 0 && row < m1) store_as(p.Out, p.outtype, row * p.ldout + t, old[k] + v);
        }
        load_u(m + (long long)AHEAD * per_pass);
    }
    cluster.barrier_wait();  // the others have read this block's sums
}

// ------------------------------------------------------------------ gradients of the factors
//
// A cluster of up to 8 blocks takes 128 rows j of Z and one adapter; its blocks share the chunks of 32 columns that hold any
// of the adapter's, in turn.  A block takes Z's and S's chunks through a ring in shared memory; a warp takes 16 rows and all
// R of S.  Columns of other adapters count as zeros in both operands (an infinity there meets a zero nowhere).
// The blocks' sums are joined through distributed shared memory in a fixed order.  Both products of a backward pass are one
// launch, dU first: it may start while dX is still being made.  Measured: K = M = 2048, 4096 columns, rank 32, three adapters,
// bf16 beside fp32 dY: 52 us for both after dX (50 MB); dU alone, both of whose operands are split, 37 us (23 us when they were
// rounded to TF32).  The splits take as many issue slots as the rest: 45% of the active cycles are busy, the tensor pipe 20%.
constexpr int GRAD_ROWS = 128;
constexpr int GRAD_CHUNK = 32;
constexpr int GRAD_SCAN = 128;  // chunks looked over at once

template <int RT>
struct GradShape {
    static constexpr int RP = RT * 16;
    static constexpr int PITCH = GRAD_CHUNK * 4 + 16;  // bytes of a chunk's row (16-bit rows use a part)
    static constexpr int STAGE = (GRAD_ROWS + RP) * PITCH;
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
    __shared__ unsigned members[GRAD_SCAN];  // which columns of a chunk are the adapter's
    __shared__ unsigned char list[GRAD_SCAN];
    __shared__ int count, seen;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long t_end = w.N;

    // A thread's 16-byte pieces of a chunk lie in rows first + k * (256 / CH), one column.
    constexpr int PER = 16 / (int)sizeof(TZ), CH = GRAD_CHUNK / PER;
    const int z_row = threadIdx.x / CH, z_col = threadIdx.x % CH * PER, s_row = threadIdx.x / 8, s_col = threadIdx.x % 8 * 4;
    const TZ *const z_src = (const TZ *)p.Z + (j0 + z_row) * p.ldz + z_col;
    const long long s_ld = Hidden::pitch_of(w.N);
    const float *const s_src = p.S + s_row * s_ld + s_col;
    const int j_left = (int)min((long long)GRAD_ROWS, p.n - j0);
    auto fill = [&](int slot, long long t0) {
        unsigned char *z = smem + slot * Q::STAGE, *s = z + GRAD_ROWS * Q::PITCH;
        const int cols = (int)min((long long)GRAD_CHUNK, t_end - t0);
        if (p.vec) {
            const int left = cols - z_col, bytes = left <= 0 ? 0 : left >= PER ? 16 : left * (int)sizeof(TZ);
#pragma unroll
            for (int k = 0; k < GRAD_ROWS * CH / 256; ++k) {
                constexpr int RS = 256 / CH;
                const int valid = z_row + k * RS < j_left ? bytes : 0;
                copy16(z + (z_row + k * RS) * Q::PITCH + z_col * (int)sizeof(TZ), valid ? z_src + t0 + k * RS * p.ldz : (const TZ *)p.Z, valid);
            }
        } else {
            copy_loose<TZ, GRAD_ROWS, GRAD_CHUNK, Q::PITCH, 256, 4>(z, (const TZ *)p.Z + j0 * p.ldz + t0, p.ldz, j_left, cols, p.word, threadIdx.x);
        }
        const int left = cols - s_col, bytes = left <= 0 ? 0 : left >= 4 ? 16 : left * 4;
#pragma unroll
        for (int k = 0; k < (Q::RP * 8 + 255) / 256; ++k) {
            const int valid = s_row + k * 32 < w.R ? bytes : 0;
            if (Q::RP >= 32 || s_row < Q::RP)
                copy16(s + (s_row + k * 32) * Q::PITCH + s_col * 4, valid ? s_src + t0 + k * 32 * s_ld : p.S, valid);
        }
    };

    if (threadIdx.x == 0) seen = 0;
    for (long long scan = 0; scan < t_end; scan += GRAD_SCAN * GRAD_CHUNK) {
        __syncthreads();
        int id[GRAD_SCAN / 8];
        w.c.of(scan + warp * GRAD_CHUNK + lane, 8 * GRAD_CHUNK, t_end, id);
#pragma unroll
        for (int k = 0; k < GRAD_SCAN / 8; ++k) {
            // Columns past the end are read as zeros: they may count as the adapter's.
            const bool any = __any_sync(~0u, id[k] == a);
            const unsigned m = __ballot_sync(~0u, id[k] == a || id[k] == -2);
            if (lane == 0) members[warp + k * 8] = any ? m : 0u;
        }
        __syncthreads();
        if (warp == 0) {
            int n = 0, all = seen;
#pragma unroll
            for (int k = lane; k < GRAD_SCAN; k += 32) {
                const bool any = members[k] != 0u;
                const unsigned m = __ballot_sync(~0u, any), before = m & ((1u << lane) - 1);
                // Every ranks-th chunk of the adapter's, over all scans, is this block's.
                const bool own = any && (all + __popc(before)) % ranks == rank;
                const unsigned o = __ballot_sync(~0u, own);
                if (own) list[n + __popc(o & ((1u << lane) - 1))] = (unsigned char)k;
                n += __popc(o);
                all += __popc(m);
            }
            __syncwarp();
            if (lane == 0) {
                count = n;
                seen = all;
            }
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
            const unsigned member = members[list[i]];
            const auto multiply = [&](auto mixed) {
#pragma unroll
                for (int k = 0; k < GRAD_CHUNK; k += 8) {
                    const bool in[2] = {!mixed.value || (member >> (k + q) & 1), !mixed.value || (member >> (k + q + 4) & 1)};
                    Operand<IS_SPLIT<TZ>> A[4];
                    TZ u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        u[e] = *(const TZ *)(z + (g + (e & 1) * 8) * Q::PITCH + (k + q + (e >> 1) * 4) * sizeof(TZ));
                        if (!in[e >> 1]) u[e] = from_float<TZ>(0.0f);
                    }
                    operands(u, A);
#pragma unroll
                    for (int b = 0; b < RT * 2; ++b) {
                        Operand<true> B[2];
                        float v[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            v[e] = *(const float *)(s + (b * 8 + g) * Q::PITCH + (k + q + e * 4) * 4);
                            if (!in[e]) v[e] = 0.0f;
                        }
                        operands<IS_SPLIT<TZ>>(v, B);
                        if constexpr (sizeof(TF) == 4) {  // long sums are kept outside the tensor cores, which cut them
                            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma8_any(part, A, B);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[b][e] += part[e];
                        } else {
                            mma8_any(acc[b], A, B);
                        }
                    }
                }
            };
            if (member == ~0u)
                multiply(std::false_type{});
            else
                multiply(std::true_type{});
        }
        copy_wait<0>();
    }
}

template <typename TF, int RT>
__global__ void __launch_bounds__(256, RT <= 4 ? 2 : 0) lora_grad(const GradParams w)
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
    // The first product's S was there before the kernel ahead of this one; the second's was made just before that one, and
    // nothing may come after this kernel while one ahead of it still runs.
    if (second) cudaGridDependencySynchronize();
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
        // Each block joins its share of the rows, in place (nobody else reads them), and writes them out.
        const int own = GRAD_ROWS / ranks;
        for (int i = threadIdx.x; i < own * Q::RP; i += 256) {
            const int at = (rank * own + i / Q::RP) * Q::SUM_PITCH + i % Q::RP;
            float x[8], v = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = k < ranks ? cluster.map_shared_rank(sum, k)[at] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v += x[k];
            sum[at] = v;
        }
        __syncthreads();
        TF *G = (TF *)p.G + (long long)a * p.n * w.R;
        for (int i = threadIdx.x; i < own * w.R; i += 256) {
            // Neighbouring threads write neighbouring elements.
            const int r = p.gr == 1 ? i % w.R : i / own, j = rank * own + (p.gr == 1 ? i / w.R : i % own);
            if (j0 + j < p.n) G[(j0 + j) * p.gj + r * p.gr] = from_float<TF>(sum[j * Q::SUM_PITCH + r]);
        }
        cluster.sync();
    }
    if (!second) cudaGridDependencySynchronize();
}

// ------------------------------------------------------------------ launches
// A launch in clusters of `ranks` blocks (0: none) that may (`early`) start before the kernel ahead of it has ended.
template <typename... Args>
tcaspmm_status launch(const char *what, void (*kernel)(Args...), dim3 grid, int ranks, bool early, int shared, cudaStream_t st, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    if (ranks) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = (unsigned)ranks;
        at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (early) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = at;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? TCASPMM_OK : cuda_fail(e, what);
}

// Allows a kernel `shared` bytes of dynamic shared memory on the current device; `done` is the kernel's, a bit a device.
inline tcaspmm_status allow_shared(const char *what, const void *kernel, int shared, std::atomic<unsigned long long> &done)
{
    int dev = 0;
    if (shared <= 48 * 1024 || (cudaGetDevice(&dev) == cudaSuccess && dev < 64 && (done.load() >> dev & 1))) return TCASPMM_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
    if (e != cudaSuccess) return cuda_fail(e, what);
    if (dev < 64) done.fetch_or(1ull << dev);
    return TCASPMM_OK;
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

// Columns of a tile of the first product: a warp's sums (RT x TN / 8 x 4 registers a thread) take at most 128 registers.
constexpr int tile_columns(int rt) { return rt <= 4 ? 64 : rt == 8 ? 32 : 16; }

template <typename TF, typename TI, bool TRANS>
tcaspmm_status shrink(ApplyParams p, int sms, cudaStream_t st)
{
    return with_rank(p.R, [&](auto rt) {
        constexpr int RT = rt.value, TN = tile_columns(RT);
        using Q = ShrinkShape<TF, TI, RT, TN, TRANS>;
        const auto kernel = lora_shrink<TF, TI, RT, TN, TRANS>;
        const long long tiles = ceil_div(p.N, TN);
        // Idle SMs take a share, while a warp has a step to do: at most one wave of blocks.
        int ranks = 1;
        while (ranks < 8 && tiles * ranks * 2 <= Q::BLOCKS * sms && p.n1 > (long long)ranks * WARPS * Q::KS) ranks *= 2;
        p.per1 = ceil_div(ceil_div(p.n1, ranks), Q::KS) * Q::KS;
        if (tiles * ranks > INT_MAX) return fail(TCASPMM_ERR_UNSUPPORTED, "lora: too many columns");
        static std::atomic<unsigned long long> done{0};
        const tcaspmm_status s = allow_shared("lora launch", (const void *)kernel, Q::BYTES, done);
        return s != TCASPMM_OK ? s : launch("lora launch", kernel, dim3((unsigned)(tiles * ranks)), ranks, false, Q::BYTES, st, p);
    });
}

template <typename TF, bool TRANS>
tcaspmm_status expand(ApplyParams p, int sms, cudaStream_t st)
{
    return with_rank(p.R, [&](auto rt) {
        constexpr int RT = rt.value;
        using Q = ExpandShape<TF, RT, TRANS>;
        const auto kernel = lora_expand<TF, RT, TRANS>;
        const long long across = ceil_div(p.N, EXP_COLS), chunks = ceil_div(p.n2, EXP_ROWS);
        if (chunks == 0) return TCASPMM_OK;
        // As many chunks a block as leave every SM eight blocks (those with several adapters take longer).
        p.chunks = (int)std::max<long long>(1, std::min<long long>(8, across * chunks / (8 * sms)));
        const long long blocks = across * ceil_div(chunks, p.chunks);
        if (blocks > INT_MAX) return fail(TCASPMM_ERR_UNSUPPORTED, "lora: too many elements");
        static std::atomic<unsigned long long> done{0};
        const tcaspmm_status s = allow_shared("lora launch", (const void *)kernel, Q::BYTES, done);
        return s != TCASPMM_OK ? s : launch("lora launch", kernel, dim3((unsigned)blocks), 0, true, Q::BYTES, st, p);
    });
}

// Where the forward pass goes column by column: up to 64 columns, or 256 where tiles of 64 may hold many adapters, within the
// work that its reads of the factors from L2 are worth.  Measured (fp16, columns one by one against tiles): 64 columns of 64
// adapters of rank 16, 4096 x 1024: 9 and 61 us, 256 of them 29 and 80; 64 columns of rank 64, 4096 x 4096, 8 adapters: 40 and
// 56 us, 128 of them more than 80 and 56; 64 columns of rank 8, 512 x 512, one adapter: 6.2 and 7.7 us, 128 of them 10.8 and 7.5.
// fp32, whose tiles take longer still: 64 columns of 64 adapters of rank 16, 4096 x 1024: 11 and 132 us; 64 of rank 64,
// 5120 x 5120, 8 adapters: 41 and 194 us, one adapter: 40 and 40 us; 256 columns of 16 adapters of rank 16, 4096 x 2048: 39 and
// 107 us.
inline bool by_token(long long L, long long R, long long M, long long K, long long N)
{
    if (N > 256 || K > 8ll * 8192) return false;
    const long long work = N * R * (K + M);
    return (N <= 64 ? work <= 40ll << 20 : L >= 16 && work <= 24ll << 20);
}

template <typename TF>
tcaspmm_status token(ApplyParams p, cudaStream_t st)
{
    constexpr int VEC = 16 / (int)sizeof(TF);
    p.per1 = ceil_div(ceil_div(p.n1, TOKEN_RANKS), VEC) * VEC;
    const int shared = (int)std::max<long long>(p.per1, 1) * 4;
    const dim3 grid((unsigned)(p.N * TOKEN_RANKS));
    if (p.vec_f1 && p.vec_f2) return launch("lora launch", lora_token<TF, VEC, VEC>, grid, TOKEN_RANKS, false, shared, st, p);
    if (p.vec_f1) return launch("lora launch", lora_token<TF, VEC, 1>, grid, TOKEN_RANKS, false, shared, st, p);
    if (p.vec_f2) return launch("lora launch", lora_token<TF, 1, VEC>, grid, TOKEN_RANKS, false, shared, st, p);
    return launch("lora launch", lora_token<TF, 1, 1>, grid, TOKEN_RANKS, false, shared, st, p);
}

template <typename TF, typename TI, bool TRANS>
tcaspmm_status apply(const ApplyParams &p, int sms, cudaStream_t st)
{
    const tcaspmm_status s = shrink<TF, TI, TRANS>(p, sms, st);
    return s != TCASPMM_OK || !p.Out ? s : expand<TF, TRANS>(p, sms, st);
}

template <typename TF>
tcaspmm_status grads(GradParams w, bool early, int sms, cudaStream_t st)
{
    return with_rank(w.R, [&](auto rt) {
        constexpr int RT = rt.value;
        const auto kernel = lora_grad<TF, RT>;
        for (GradProblem &p : w.p) p.tiles = p.G ? (int)ceil_div(p.n, GRAD_ROWS) : 0;
        const long long tiles = (long long)w.p[0].tiles + w.p[1].tiles;
        if (tiles == 0 || w.c.L == 0) return TCASPMM_OK;
        int ranks = 1;
        while (ranks < 8 && tiles * ranks < 2 * sms && w.N > (long long)ranks * 2 * GRAD_CHUNK) ranks *= 2;
        if (tiles * ranks > INT_MAX) return fail(TCASPMM_ERR_UNSUPPORTED, "lora_backward: too many rows");
        static std::atomic<unsigned long long> done{0};
        const tcaspmm_status s = allow_shared("lora_backward launch", (const void *)kernel, GradShape<RT>::BYTES, done);
        return s != TCASPMM_OK ? s
                               : launch("lora_backward launch", kernel, dim3((unsigned)(tiles * ranks), (unsigned)std::min(w.c.L, 65535)),
                                        ranks, early, GradShape<RT>::BYTES, st, w);
    });
}

}  // namespace
}  // namespace tca
