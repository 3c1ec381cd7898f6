// Shared parts of layer norm (norm.cu, norm_grad.cuh): the mathematics, the split of the work, launches.
//
// Layer norm, forward and backward, over the rows' elements (dim 1: a node's features, the layout of a graph product's C)
// or the columns' (dim 0: a token's features, the layout of a pruned weight's B).
//
//   mean = sum x / n    rstd = 1 / sqrt(sum (x - mean)^2 / n + eps)    xh = (x - mean) rstd    y = w xh + b
//   g = w dy            dx = rstd (g - mean(g) - xh mean(g xh))        dw = sum dy xh          db = sum dy
//
// Every pass is bound by memory: the vector is read once, held as it came (registers, or shared memory), and summed twice there
// (the mean first, then the squared differences from it, so that a large mean costs no precision).  Rows: a part of a warp, a
// warp or a block per row, whichever leaves a thread at most 16 elements.  Columns: a cluster of up to 8 blocks shares a strip
// of 16-64 columns, each block holds a part of the strip's rows, and the blocks exchange their sums through distributed shared
// memory, so that reads stay coalesced along the rows.  The weight's gradient is summed by each thread over the vectors it
// meets (its features stay the same), by block through shared memory, and over the blocks by a second kernel, in a fixed order.
//
// Measured (one B200, whose copy of large arrays reaches 6.5 TB/s): rows, 2^20 x 128 fp32, forward 167 us (6.4 TB/s), backward
// 258 us (6.2 TB/s); 4096 x 8192 bf16, forward 40 us, backward 65 us; 100003 x 233 fp32 to bf16, whose rows allow no vectors,
// 36 us (3.9 TB/s; about two thirds of the issue slots busy).  Columns, 4096 x 8192 bf16, forward 42 us (3.2 TB/s), backward
// 82 us (2.5 TB/s): there the sums, the exchange between blocks and the unpacking of 16-bit elements take as long as memory.
// Wide rows leave a thread 64 registers, which is too few: the backward kernels of 8193 to 16384 elements spill 160 to 376 bytes a
// thread, with one element a load 464 to 856, and with one element a load the forward kernel spills 168 to 196 from 2049 on.
// 4096 x 16384 bf16: forward 81 us, backward 159 us; 4096 x 16383: 420 and 1250 us; 4096 x 8191: 196 and 158 us.  Rows past
// 16384 elements are read two or three times, element by element: 4096 x 20000 bf16, 450 and 1100 us.
#pragma once

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstring>
#include <type_traits>

#include <cooperative_groups.h>

#include "dense.h"

namespace cg = cooperative_groups;

namespace tca {

int sm_count();  // SMs of the current device (norm.cu)

struct NormParams {
    const void *X;
    long long ldx;
    void *Y;
    long long ldy;
    int yt;
    const void *w, *b;  // one per feature, type pt, or NULL
    int pt;
    int pvec;            // w and b allow vector loads
    float *mean, *rstd;  // one per vector, or NULL
    long long vecs, n;   // vectors normalised, their length
    float eps;
};

struct NormGradParams {
    const void *dY;
    long long lddy;
    int dyt;
    const void *X;
    long long ldx;
    const float *mean, *rstd;
    const void *w;
    int pt;
    int pvec;
    void *dX;  // or NULL
    long long lddx;
    float *part;  // partial weight (then bias) gradients, one row of n per part, or NULL
    long long vecs, n;
};

namespace {

template <int VEC, typename T>
__device__ __forceinline__ void store_pack(T *p, const float (&v)[VEC])
{
    constexpr int PER = sizeof(T) * VEC > 16 ? 16 / (int)sizeof(T) : VEC;
#pragma unroll
    for (int k = 0; k < VEC; k += PER) {
        T t[PER];
        if constexpr (sizeof(T) == 2 && PER % 2 == 0) {
#pragma unroll
            for (int i = 0; i < PER; i += 2) {  // two at a time: one conversion instruction
                if constexpr (std::is_same<T, __half>::value) {
                    const __half2 two = __floats2half2_rn(v[k + i], v[k + i + 1]);
                    memcpy(t + i, &two, 4);
                } else {
                    const __nv_bfloat162 two = __floats2bfloat162_rn(v[k + i], v[k + i + 1]);
                    memcpy(t + i, &two, 4);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) t[i] = from_float<T>(v[k + i]);
        }
        typename Bits<sizeof(T) * PER>::type bits;
        memcpy(&bits, t, sizeof bits);
        *reinterpret_cast<decltype(bits) *>(p + k) = bits;
    }
}

// VEC elements in shared memory.
template <typename T, int VEC>
__device__ __forceinline__ void load_shared(const T *p, float *v)
{
    Pack<T, VEC> t;
    t.bits = *reinterpret_cast<const decltype(t.bits) *>(p);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = t.get(e);
}

// Calls f with a value of the type of code `type`: the same branch for every thread.
template <typename F>
__device__ __forceinline__ void by_type(int type, F &&f)
{
    if (type == 0)
        f(float{});
    else if (type == 1)
        f(__half{});
    else
        f(__nv_bfloat16{});
}

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T *p, float *v)
{
    constexpr int PER = sizeof(T) * VEC > 16 ? 16 / (int)sizeof(T) : VEC;
#pragma unroll
    for (int k = 0; k < VEC; k += PER) {
        Pack<T, PER> t;
        t.load(p + k);
#pragma unroll
        for (int i = 0; i < PER; ++i) v[k + i] = t.get(i);
    }
}

// Parameters i .. i + VEC - 1; `dflt` without a parameter.
template <int VEC>
__device__ __forceinline__ void load_params(const void *p, int type, int pvec, long long i, float dflt, float *v)
{
    if (!p) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = dflt;
    } else if (!pvec) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = load_as(p, type, i + k);
    } else if (type == 0) {
        load_pack<float, VEC>((const float *)p + i, v);
    } else if (type == 1) {
        load_pack<__half, VEC>((const __half *)p + i, v);
    } else {
        load_pack<__nv_bfloat16, VEC>((const __nv_bfloat16 *)p + i, v);
    }
}

// ------------------------------------------------------------------ rows
// Sum over a row's threads: `lanes` neighbours of a warp, or (BLOCK) the whole block through `s`, a float per warp.  Calls
// alternate between two such arrays, so one barrier a call is enough.
template <bool BLOCK, int COUNT>
__device__ __forceinline__ void row_sum(float (&v)[COUNT], int lanes, float (*s)[32])
{
#pragma unroll
    for (int o = 16; o; o >>= 1)
        if (BLOCK || o < lanes) {
#pragma unroll
            for (int k = 0; k < COUNT; ++k) v[k] += __shfl_xor_sync(~0u, v[k], o);
        }
    if (BLOCK) {
        const int warps = (int)(blockDim.x >> 5), lane = threadIdx.x & 31;
#pragma unroll
        for (int k = 0; k < COUNT; ++k)
            if (lane == 0) s[k][threadIdx.x >> 5] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < COUNT; ++k) {
            float t = lane < warps ? s[k][lane] : 0.0f;
#pragma unroll
            for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
            v[k] = t;
        }
    }
}

// ------------------------------------------------------------------ columns
//
// A cluster's block holds its part of a strip's rows in shared memory (asynchronous copies where the rows' alignment allows
// them, 16 bytes a thread), so that several blocks an SM load, sum and write at the same time: three of 64 KB.  The same
// strips in registers, one block of 512 threads an SM, took 103 us forward and 123 us backward on 4096 x 8192 bf16 (42 and 82
// here), for want of bytes on their way while a block was summing.
constexpr int STRIP_THREADS = 256;
constexpr int STRIP_WARPS = STRIP_THREADS / 32;
constexpr int STRIP_MAX = 64;  // columns of a strip at most

struct Strip {
    int lpr, shift;  // threads along a row of the strip (a power of two), its logarithm
    int per_block;   // rows of a block
};

__device__ __forceinline__ void copy_async(void *dst, const void *src, int bytes)  // 8 or 16
{
    const unsigned to = (unsigned)__cvta_generic_to_shared(dst);
    if (bytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory"); }

// Rows r0 .. r0 + rows - 1 of the strip of `width` columns (a power of two) from column c0 on, into `tile` ([row][width]); columns
// past `cols` as zeros.  Every thread's copies have landed when it returns; the block's, after a barrier.
template <typename T, int VEC>
__device__ __forceinline__ void load_strip(T *tile, const T *X, long long ld, long long r0, int rows, long long c0, long long cols, int width,
                                           const Strip &q, bool vec)
{
    if (vec) {
        const int c = (threadIdx.x & (q.lpr - 1)) * VEC;
        const T *src = X + (r0 + (threadIdx.x >> q.shift)) * ld + c0 + c;
        const long long step = (long long)(STRIP_THREADS >> q.shift) * ld;
        if (c0 + c < cols) {
            for (int r = threadIdx.x >> q.shift; r < rows; r += STRIP_THREADS >> q.shift, src += step)
                copy_async(tile + r * width + c, src, VEC * (int)sizeof(T));
        } else {
            for (int r = threadIdx.x >> q.shift; r < rows; r += STRIP_THREADS >> q.shift)
#pragma unroll
                for (int e = 0; e < VEC; ++e) tile[r * width + c + e] = from_float<T>(0.0f);
        }
    } else {
        // Element by element: a column for each thread along a row, eight rows in flight.
        const int c = threadIdx.x & (width - 1), per = STRIP_THREADS / width;
        const bool in = c0 + c < cols;
        const T *src = X + c0 + c;
        for (int r = threadIdx.x / width; r < rows; r += 8 * per) {
            T v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = in && r + k * per < rows ? src[(r0 + r + k * per) * ld] : from_float<T>(0.0f);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (r + k * per < rows) tile[(r + k * per) * width + c] = v[k];
        }
    }
}

// Sums over the block's rows of COUNT values for each of a thread's VEC columns, into `out`, one per column of the strip.
// Threads of a warp whose numbers agree modulo `lpr` hold the same columns.
template <int COUNT, int VEC>
__device__ __forceinline__ void strip_sum(float (&v)[COUNT][VEC], int lpr, float (*s)[STRIP_WARPS][STRIP_MAX], float (*out)[STRIP_MAX])
{
#pragma unroll
    for (int o = 16; o; o >>= 1)
        if (o >= lpr) {
#pragma unroll
            for (int k = 0; k < COUNT; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] += __shfl_xor_sync(~0u, v[k][e], o);
        }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane < lpr) {
#pragma unroll
        for (int k = 0; k < COUNT; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[k][warp][lane * VEC + e] = v[k][e];
    }
    __syncthreads();
    const int width = lpr * VEC;
    for (int j = threadIdx.x; j < COUNT * width; j += STRIP_THREADS) {
        const int k = j / width, c = j - k * width;
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < STRIP_WARPS; ++i) t += s[k][i][c];
        out[k][c] = t;
    }
    __syncthreads();
}

// ------------------------------------------------------------------ vectors of any length
// Sum over the block's threads, the same in all of them.  `s` holds a float per warp.
__device__ float block_sum(float v, float *s)
{
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    const int warps = blockDim.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < warps; ++i) t += s[i];
    return t;
}

// ------------------------------------------------------------------ launches
unsigned blocks_of(long long n) { return (unsigned)std::min<long long>(n, INT_MAX); }
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

tcaspmm_status launched(const char *what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TCASPMM_OK : cuda_fail(e, what);
}

// Rows of `n` elements start where VEC-element loads and stores (at most 16 bytes each) may.
bool aligned(const void *p, long long ld, int type, int vec)
{
    const int bytes = std::min(16, vec * size_of(type));
    return !p || ((uintptr_t)p % bytes == 0 && ld * size_of(type) % bytes == 0);
}

// How rows of n elements are dealt to threads: `nch` chunks of vec elements for each of `lanes` threads of a warp, or of the
// `threads` of a block (lanes 0).  nch 0: too long.
struct RowPlan {
    int nch, lanes, threads;
};

// A warp takes a row of up to 32 x `most` elements, below that the smallest power of two of lanes; a block longer ones.
RowPlan plan_rows(long long n, int vec, int most, int threads_most)
{
    const long long chunks = ceil_div(n, vec);
    const int cap = most / vec;
    if (chunks <= 32 * cap) {
        int lanes = 1;
        while (lanes < 32 && lanes < chunks) lanes *= 2;
        int nch = 1;
        while ((long long)nch * lanes < chunks) nch *= 2;
        return {nch, lanes, 256};
    }
    if (chunks > (long long)threads_most * cap) return {0, 0, 0};
    int nch = cap;
    while (nch > 1 && ceil_div(chunks, nch / 2) <= 256) nch /= 2;
    return {nch, 0, (int)(ceil_div(ceil_div(chunks, nch), 32) * 32)};
}

// How columns are dealt to clusters: strips of lpr x vec columns, `ranks` blocks a strip.  ranks 0: too long.
struct StripPlan {
    int ranks;
    Strip q;
    long long strips;
    int shared;
};

// Strips `bytes` wide (of the widest of the arrays, `size` bytes an element; `row` bytes an element over all arrays and `more`
// a row), narrower for fewer columns, and for columns that 8 blocks cannot hold in MOST bytes each.
StripPlan plan_strips(long long n, long long vecs, int vec, int size, int row, int more, int bytes, int sms)
{
    constexpr long long GOOD = 66 * 1024, MOST = 199 * 1024;  // three blocks an SM, one
    int lpr = bytes / size / vec;
    while (lpr > 1 && (lpr / 2) * vec >= vecs) lpr /= 2;
    const auto per_row = [&] { return (long long)lpr * vec * row + more; };
    while (lpr > 1 && n * per_row() > 8 * MOST) lpr /= 2;
    if (n * per_row() > 8 * MOST) return {};
    const long long strips = ceil_div(vecs, (long long)lpr * vec);
    int ranks = 1;
    while (ranks < 8 && ceil_div(n, ranks) * per_row() > GOOD) ranks *= 2;
    while (ranks < 8 && strips * ranks < sms && n > (long long)ranks * (STRIP_THREADS / lpr)) ranks *= 2;  // idle SMs take a share
    const long long per = ceil_div(n, ranks);
    if (per * per_row() > MOST) return {};
    int shift = 0;
    while ((1 << shift) < lpr) ++shift;
    return {ranks, {lpr, shift, (int)per}, strips, (int)(per * per_row()) + 32};  // the second array begins at 16 bytes
}

template <typename... Args>
tcaspmm_status launch_cluster(void (*kernel)(Args...), const StripPlan &s, std::atomic<unsigned long long> &done, cudaStream_t st, Args... args)
{
    int dev = 0;
    // More than the usual shared memory, allowed once a device.
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || !(done.load() >> dev & 1)) {
        const cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (e != cudaSuccess) return cuda_fail(e, "layer_norm launch");
        if (dev < 64) done.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(s.strips * s.ranks));
    cfg.blockDim = dim3(STRIP_THREADS);
    cfg.dynamicSmemBytes = (size_t)s.shared;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)s.ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? TCASPMM_OK : cuda_fail(e, "layer_norm launch");
}

// Blocks of `threads` threads an SM holds of a kernel (asked once: `known` is the kernel's).
inline int resident(const void *kernel, int threads, int shared, std::atomic<int> &known)
{
    int n = known.load();
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, shared) != cudaSuccess || n < 1) n = 1;
        known.store(n);
    }
    return n;
}

// Calls f with the compile-time chunk count.
template <int MOST, typename F>
tcaspmm_status with_chunks(int nch, F &&f)
{
    if (nch <= 1) return f(std::integral_constant<int, 1>{});
    if constexpr (MOST >= 2)
        if (nch == 2) return f(std::integral_constant<int, 2>{});
    if constexpr (MOST >= 4)
        if (nch == 4) return f(std::integral_constant<int, 4>{});
    if constexpr (MOST >= 8)
        if (nch == 8) return f(std::integral_constant<int, 8>{});
    if constexpr (MOST >= 16)
        if (nch == 16) return f(std::integral_constant<int, 16>{});
    if constexpr (MOST >= 32)
        if (nch == 32) return f(std::integral_constant<int, 32>{});
    return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: no kernel for %d chunks", nch);
}

constexpr int FWD_MOST = 16;       // elements of a row a thread holds, forward
constexpr int BWD_MOST = 16;       // backward, where the sums of both gradients sit beside them

// Parts the weight gradient's sums come in: blocks of the backward kernel over rows, strips over columns.
constexpr int ROW_PARTS = 4;
constexpr int LONG_PARTS = 64;

}  // namespace
}  // namespace tca
