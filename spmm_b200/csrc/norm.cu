// Layer norm: the forward kernels, the join of the weight gradient's parts and the C entries.
#include <cmath>
#include <mutex>

#include "norm.cuh"

namespace tca {

tcaspmm_status norm_backward_f32(const NormGradParams &p, int dim, long long *parts, cudaStream_t st);
tcaspmm_status norm_backward_f16(const NormGradParams &p, int dim, long long *parts, cudaStream_t st);
tcaspmm_status norm_backward_bf16(const NormGradParams &p, int dim, long long *parts, cudaStream_t st);

// SMs of the current device, 148 when it cannot be asked.
int sm_count()
{
    static std::mutex mu;
    static int known[64] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    std::lock_guard<std::mutex> lk(mu);
    if (!known[dev] && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev] = n;
    return known[dev] ? known[dev] : 148;
}

namespace {

// A row's elements are dealt to its threads VEC at a time, NCH times; a thread's elements are the same in every row.  Short rows
// go ROWS at a time, so that enough bytes are on their way; the next rows are fetched before the present ones are summed.
// LANES: threads a row, where they are a whole warp; 0: `lanes` of one, or (BLOCK) the block.
template <typename T, int VEC, int NCH, int ROWS, int LANES, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) norm_rows_fwd(const NormParams p, int lanes)
{
    constexpr bool KEEP = VEC * NCH <= 8;  // weights stay in registers
    __shared__ float s[2][ROWS][32];
    const int n = (int)p.n;
    if (LANES) lanes = LANES;
    const int tpr = BLOCK ? (int)blockDim.x : lanes;
    const int t = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1));
    const int per = BLOCK ? 1 : 256 / lanes;  // rows side by side in a block
    const long long first = (long long)blockIdx.x * per * ROWS + (BLOCK ? 0 : (int)threadIdx.x / lanes);
    const long long step = (long long)gridDim.x * per * ROWS;
    const float inv = 1.0f / (float)n;
    float w[KEEP ? VEC * NCH : 1], b[KEEP ? VEC * NCH : 1];
    if (KEEP) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int i = (c * tpr + t) * VEC;
            if (i < n) {
                load_params<VEC>(p.w, p.pt, p.pvec, i, 1.0f, w + c * VEC);
                load_params<VEC>(p.b, p.pt, p.pvec, i, 0.0f, b + c * VEC);
            }
        }
    }
    Pack<T, VEC> x[ROWS][NCH], next[ROWS][NCH];
    auto fetch = [&](long long row, Pack<T, VEC> (&to)[ROWS][NCH]) {  // rows row, row + per, ...
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const bool in = row + r * per < p.vecs;
            const T *src = (const T *)p.X + (row + r * per) * p.ldx + t * VEC;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                if (in && (c * tpr + t) * VEC < n)
                    to[r][c].load(src + c * tpr * VEC);
                else
                    to[r][c].zero();
            }
        }
    };
    fetch(first, x);
    // Every thread of a warp (block) takes the same number of turns: rows past the end are read as zeros and not written.
    for (long long start = (long long)blockIdx.x * per * ROWS, row = first; start < p.vecs; start += step, row += step) {
        fetch(row + step, next);
        float mean[ROWS], sq[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            mean[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) mean[r] += x[r][c].get(e);
        }
        row_sum<BLOCK>(mean, lanes, s[0]);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            mean[r] *= inv;
            sq[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
                if ((c * tpr + t) * VEC < n) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float d = x[r][c].get(e) - mean[r];
                        sq[r] += d * d;
                    }
                }
        }
        row_sum<BLOCK>(sq, lanes, s[1]);
        by_type(p.yt, [&](auto type) {
            using TO = decltype(type);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const long long at = row + r * per;
                if (at >= p.vecs) continue;
                const float rstd = 1.0f / sqrtf(sq[r] * inv + p.eps);
                TO *const out = (TO *)p.Y + at * p.ldy + t * VEC;
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    const int i = (c * tpr + t) * VEC;
                    if (i < n) {
                        float y[VEC], ww[VEC], bb[VEC];
                        if (!KEEP) {
                            load_params<VEC>(p.w, p.pt, p.pvec, i, 1.0f, ww);
                            load_params<VEC>(p.b, p.pt, p.pvec, i, 0.0f, bb);
                        }
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            y[e] = fmaf((x[r][c].get(e) - mean[r]) * rstd, KEEP ? w[c * VEC + e] : ww[e], KEEP ? b[c * VEC + e] : bb[e]);
                        store_pack<VEC>(out + c * tpr * VEC, y);
                    }
                }
                if (t == 0 && p.mean) {
                    p.mean[at] = mean[r];
                    p.rstd[at] = rstd;
                }
            }
        });
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int c = 0; c < NCH; ++c) x[r][c] = next[r][c];
    }
}

template <typename T>
__global__ void __launch_bounds__(STRIP_THREADS) norm_cols_fwd(const NormParams p, const Strip q, int vec)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float s[1][STRIP_WARPS][STRIP_MAX];
    __shared__ float sums[2][STRIP_MAX];  // this block's sum of x, then of squared differences from its own mean
    __shared__ __align__(16) float fin[2][STRIP_MAX];  // the strip's mean and rstd
    T *const tile = (T *)smem;
    float2 *const wb = (float2 *)(smem + ((size_t)q.per_block * (q.lpr * VEC) * sizeof(T) + 15) / 16 * 16);  // the rows' weight and bias
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int width = q.lpr * VEC, at = (threadIdx.x & (q.lpr - 1)) * VEC;
    const long long c0 = (long long)(blockIdx.x / ranks) * width;
    const long long r0 = min(p.n, (long long)rank * q.per_block);
    const int rows = (int)(min(p.n, r0 + q.per_block) - r0);
    const int row = threadIdx.x >> q.shift, step = STRIP_THREADS >> q.shift;
    load_strip<T, VEC>(tile, (const T *)p.X, p.ldx, r0, rows, c0, p.vecs, width, q, vec);
    for (int r = threadIdx.x; r < rows; r += STRIP_THREADS)
        wb[r] = make_float2(p.w ? load_as(p.w, p.pt, r0 + r) : 1.0f, p.b ? load_as(p.b, p.pt, r0 + r) : 0.0f);
    copy_async_wait();
    __syncthreads();
    float v[1][VEC] = {};
#pragma unroll 4
    for (int r = row; r < rows; r += step) {
        float x[VEC];
        load_shared<T, VEC>(tile + r * width + at, x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[0][e] += x[e];
    }
    strip_sum(v, q.lpr, s, sums);
    const float inv = rows > 0 ? 1.0f / (float)rows : 0.0f;
    float m[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        m[e] = sums[0][at + e] * inv;
        v[0][e] = 0.0f;
    }
#pragma unroll 4
    for (int r = row; r < rows; r += step) {
        float x[VEC];
        load_shared<T, VEC>(tile + r * width + at, x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = x[e] - m[e];
            v[0][e] += d * d;
        }
    }
    strip_sum(v, q.lpr, s, sums + 1);
    if (ranks > 1) cluster.sync();
    // Blocks' sums joined: sum (x - mean)^2 = sum over blocks of its own about its mean + rows (its mean - mean)^2.
    if ((int)threadIdx.x < width) {
        const int j = threadIdx.x;
        float part[8], own[8], total = 0.0f, sq = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float *o = cluster.map_shared_rank(&sums[0][0], k < ranks ? k : 0);
            part[k] = k < ranks ? o[j] : 0.0f;
            own[k] = k < ranks ? o[STRIP_MAX + j] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) total += part[k];
        const float mean = total / (float)p.n;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const long long count = k < ranks ? min(p.n, (long long)(k + 1) * q.per_block) - min(p.n, (long long)k * q.per_block) : 0;
            if (count > 0) {
                const float d = part[k] * (1.0f / (float)count) - mean;
                sq += own[k] + (float)count * d * d;
            }
        }
        fin[0][j] = mean;
        fin[1][j] = 1.0f / sqrtf(sq / (float)p.n + p.eps);
        if (p.mean && rank == 0 && c0 + j < p.vecs) {
            p.mean[c0 + j] = mean;
            p.rstd[c0 + j] = fin[1][j];
        }
    }
    __syncthreads();
    if (ranks > 1) cluster.barrier_arrive();  // this block has read the others' sums
    by_type(p.yt, [&](auto type) {
        using TO = decltype(type);
        if (vec) {
            float mean[VEC], rstd[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                mean[e] = fin[0][at + e];
                rstd[e] = fin[1][at + e];
            }
            if (c0 + at >= p.vecs) return;
            TO *out = (TO *)p.Y + (r0 + row) * p.ldy + c0 + at;
            const long long down = step * p.ldy;
#pragma unroll 4
            for (int r = row; r < rows; r += step, out += down) {
                const float2 k = wb[r];
                float x[VEC];
                load_shared<T, VEC>(tile + r * width + at, x);
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[e] = fmaf((x[e] - mean[e]) * rstd[e], k.x, k.y);
                store_pack<VEC>(out, x);
            }
        } else {
            const int c = threadIdx.x & (width - 1), per = STRIP_THREADS / width;
            const float mean = fin[0][c], rstd = fin[1][c];
            if (c0 + c >= p.vecs) return;
            TO *out = (TO *)p.Y + (r0 + threadIdx.x / width) * p.ldy + c0 + c;
            const long long down = per * p.ldy;
#pragma unroll 4
            for (int r = threadIdx.x / width; r < rows; r += per, out += down) {
                const float2 k = wb[r];
                *out = from_float<TO>(fmaf((to_float(tile[r * width + c]) - mean) * rstd, k.x, k.y));
            }
        }
    });
    if (ranks > 1) cluster.barrier_wait();
}

// One block per vector, read three times: for vectors too long for the registers of a block (rows) or a cluster (columns).
// Element i of vector v lies at v * sv + i * si.
template <typename T>
__global__ void __launch_bounds__(1024) norm_long_fwd(const NormParams p, long long sv, long long si, long long yv, long long yi)
{
    __shared__ float s[32];
    for (long long v = blockIdx.x; v < p.vecs; v += gridDim.x) {
        const T *x = (const T *)p.X + v * sv;
        float a = 0.0f;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) a += to_float(x[i * si]);
        const float mean = block_sum(a, s) / (float)p.n;
        a = 0.0f;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float d = to_float(x[i * si]) - mean;
            a += d * d;
        }
        const float rstd = 1.0f / sqrtf(block_sum(a, s) / (float)p.n + p.eps);
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float xh = (to_float(x[i * si]) - mean) * rstd;
            store_as(p.Y, p.yt, v * yv + i * yi,
                     xh * (p.w ? load_as(p.w, p.pt, i) : 1.0f) + (p.b ? load_as(p.b, p.pt, i) : 0.0f));
        }
        if (threadIdx.x == 0 && p.mean) {
            p.mean[v] = mean;
            p.rstd[v] = rstd;
        }
    }
}

// dw (y = 0) and db (y = 1): the parts of each feature added in a fixed order, 32 features a block.
__global__ void __launch_bounds__(1024) norm_join(const float *part, long long parts, long long n, void *dw, void *db, int type)
{
    __shared__ float s[32][33];
    void *out = blockIdx.y ? db : dw;
    if (!out) return;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const long long i = (long long)blockIdx.x * 32 + x;
    float a = 0.0f;
    if (i < n)
        for (long long k = y; k < parts; k += 32) a += part[(blockIdx.y * parts + k) * n + i];
    s[y][x] = a;
    __syncthreads();
    a = s[x][y];
#pragma unroll
    for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
    const long long j = (long long)blockIdx.x * 32 + y;
    if (x == 0 && j < n) store_as(out, type, j, a);
}

template <typename T, int VEC>
tcaspmm_status forward(const NormParams &p, int dim, cudaStream_t st)
{
    if (dim == 1) {
        const RowPlan r = plan_rows(p.n, VEC, FWD_MOST, 1024);
        if (r.nch) {
            return with_chunks<FWD_MOST / VEC>(r.nch, [&](auto nch) {
                constexpr int N = nch.value, ROWS = N * VEC * (int)sizeof(T) <= 16 ? 4 : N * VEC * (int)sizeof(T) <= 32 ? 2 : 1;
                // One wave of blocks, each with its share of the rows; of the shortest rows, whose weights are few, blocks of
                // four turns (2^20 x 128 fp32: 167 us, in one wave a quarter more; 2^19 x 256 fp16 the other way, a fifth more).
                const auto launch = [&](auto kernel, std::atomic<int> &known) {
                    const long long wave = (long long)resident((const void *)kernel, 256, 0, known) * sm_count();
                    const long long turns = ceil_div(p.vecs, 256 / r.lanes * ROWS);
                    const long long blocks = std::min(turns, N * VEC <= 4 ? std::max(wave, ceil_div(turns, 4)) : wave);
                    kernel<<<blocks_of(blocks), 256, 0, st>>>(p, r.lanes);
                    return launched("layer_norm launch");
                };
                if (r.lanes == 32) {
                    static std::atomic<int> known;
                    return launch(norm_rows_fwd<T, VEC, N, ROWS, 32, false>, known);
                }
                if constexpr (N == 1) {  // a part of a warp: one chunk a thread
                    if (r.lanes) {
                        static std::atomic<int> known;
                        return launch(norm_rows_fwd<T, VEC, N, ROWS, 0, false>, known);
                    }
                }
                if constexpr (N * VEC * 4 >= FWD_MOST) {  // a block: a quarter of the most, or more
                    if (!r.lanes) {
                        const long long fit = (long long)std::max(1, 1024 / r.threads) * sm_count();
                        norm_rows_fwd<T, VEC, N, 1, 0, true><<<blocks_of(std::min(p.vecs, fit)), r.threads, 0, st>>>(p, 32);
                        return launched("layer_norm launch");
                    }
                }
                return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: no kernel for rows of %lld", p.n);
            });
        }
    } else {
        const StripPlan q = plan_strips(p.n, p.vecs, 16 / (int)sizeof(T), sizeof(T), sizeof(T), 8, 128, sm_count());
        static std::atomic<unsigned long long> done{0};
        if (q.ranks && q.strips * q.ranks <= INT_MAX) return launch_cluster(norm_cols_fwd<T>, q, done, st, p, q.q, (int)(VEC > 1));
    }
    norm_long_fwd<T><<<blocks_of(p.vecs), 1024, 0, st>>>(p, dim ? p.ldx : 1, dim ? 1 : p.ldx, dim ? p.ldy : 1, dim ? 1 : p.ldy);
    return launched("layer_norm launch");
}

}  // namespace
}  // namespace tca

using namespace tca;

extern "C" tcaspmm_status tcaspmm_layer_norm(const void *dX, int64_t ldx, tcaspmm_dtype x_dt, void *dY, int64_t ldy,
                                             tcaspmm_dtype y_dt, const void *weight, const void *bias, tcaspmm_dtype p_dt,
                                             float *mean, float *rstd, int64_t rows, int64_t cols, int dim, double eps,
                                             void *stream)
{
    clear_error();
    if (!dtype_valid(x_dt) || !dtype_valid(y_dt) || !dtype_valid(p_dt))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: unknown dtype");
    if (dim != 0 && dim != 1) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: dim must be 0 or 1, not %d", dim);
    const int xt = type_code(x_dt), yt = type_code(y_dt), pt = type_code(p_dt);
    if (rows < 0 || cols < 0 || !matrix_ok(dX, rows, cols, ldx, xt) || !matrix_ok(dY, rows, cols, ldy, yt))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: bad sizes rows=%lld cols=%lld ldx=%lld ldy=%lld, NULL or misaligned pointer",
                    (long long)rows, (long long)cols, (long long)ldx, (long long)ldy);
    if (!(eps >= 0.0) || std::isinf(eps)) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: eps must be finite and not negative");
    if (!mean != !rstd) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: mean and rstd go together");
    if (!pointer_ok(weight, pt) || !pointer_ok(bias, pt) || !pointer_ok(mean, 0) || !pointer_ok(rstd, 0))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: misaligned weight, bias, mean or rstd");
    const long long vecs = dim == 1 ? rows : cols, n = dim == 1 ? cols : rows;
    if (overlaps_any(Extent(dY, rows, cols, ldy, size_of(yt)), {Extent(dX, rows, cols, ldx, size_of(xt)), Extent(weight, 1, n, n, size_of(pt)),
                                                                Extent(bias, 1, n, n, size_of(pt))}))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: Y shares memory with an input");
    if (vecs == 0) return TCASPMM_OK;
    if (n == 0) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: the normalised dimension is empty");
    NormParams p{dX, ldx, dY, ldy, yt, weight, bias, pt, 0, mean, rstd, vecs, n, (float)eps};
    return with_type(xt, [&](auto t) {
        using T = decltype(t);
        constexpr int VEC = 16 / (int)sizeof(T);
        p.pvec = aligned(weight, 0, pt, VEC) && aligned(bias, 0, pt, VEC);
        if (cols % VEC == 0 && aligned(dX, ldx, xt, VEC) && aligned(dY, ldy, yt, VEC))
            return forward<T, VEC>(p, dim, (cudaStream_t)stream);
        return forward<T, 1>(p, dim, (cudaStream_t)stream);
    });
}

extern "C" size_t tcaspmm_layer_norm_backward_workspace(int64_t rows, int64_t cols, int dim)
{
    if (rows <= 0 || cols <= 0) return 0;
    const long long n = dim == 1 ? cols : rows, vecs = dim == 1 ? rows : cols;
    // Rows: ROW_PARTS blocks an SM, or LONG_PARTS.  Columns: a strip for every 16 columns; of columns that 8 blocks' shared
    // memory holds only in narrower strips (199 KB each, at most 8 bytes an element), for every 8, 4, ...
    long long width = 16;
    while (width > 4 && (width * 8 + 4) * n > 8 * 199 * 1024) width /= 2;
    const long long parts = dim == 1 ? std::max<long long>((long long)ROW_PARTS * sm_count(), LONG_PARTS) : ceil_div(vecs, width);
    return (size_t)(2 * std::min(parts, std::max<long long>(vecs, 1)) * n) * sizeof(float);
}

extern "C" tcaspmm_status tcaspmm_layer_norm_backward(const void *dDY, int64_t lddy, tcaspmm_dtype dy_dt, const void *dX,
                                                      int64_t ldx, tcaspmm_dtype x_dt, const float *mean, const float *rstd,
                                                      const void *weight, tcaspmm_dtype p_dt, void *dDX, int64_t lddx,
                                                      void *dweight, void *dbias, int64_t rows, int64_t cols, int dim,
                                                      void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    if (!dtype_valid(x_dt) || !dtype_valid(dy_dt) || !dtype_valid(p_dt))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: unknown dtype");
    if (dim != 0 && dim != 1) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: dim must be 0 or 1, not %d", dim);
    const int xt = type_code(x_dt), gt = type_code(dy_dt), pt = type_code(p_dt);
    if (rows < 0 || cols < 0 || !matrix_ok(dX, rows, cols, ldx, xt) || !matrix_ok(dDY, rows, cols, lddy, gt) ||
        (dDX && !matrix_ok(dDX, rows, cols, lddx, xt)))
        return fail(TCASPMM_ERR_INVALID_ARG,
                    "layer_norm_backward: bad sizes rows=%lld cols=%lld ldx=%lld lddy=%lld lddx=%lld, NULL or misaligned pointer",
                    (long long)rows, (long long)cols, (long long)ldx, (long long)lddy, (long long)lddx);
    const long long vecs = dim == 1 ? rows : cols, n = dim == 1 ? cols : rows;
    if (n == 0) return vecs == 0 ? TCASPMM_OK : fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: the normalised dimension is empty");
    if (vecs > 0 && (!mean || !rstd)) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: mean and rstd are needed");
    if (!pointer_ok(mean, 0) || !pointer_ok(rstd, 0) || !pointer_ok(weight, pt) || !pointer_ok(dweight, pt) || !pointer_ok(dbias, pt))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: misaligned mean, rstd, weight, dweight or dbias");
    if (overlaps_any(Extent(dDX, rows, cols, lddx, size_of(xt)), {Extent(dX, rows, cols, ldx, size_of(xt)), Extent(dDY, rows, cols, lddy, size_of(gt)),
                                                                  Extent(weight, 1, n, n, size_of(pt))}))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: dX shares memory with an input");
    const bool params = dweight || dbias;
    const size_t need = params ? tcaspmm_layer_norm_backward_workspace(rows, cols, dim) : 0;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: a workspace of %zu bytes, 16-byte aligned, is needed", need);
    const cudaStream_t st = (cudaStream_t)stream;
    NormGradParams p{dDY, lddy, gt, dX, ldx, mean, rstd, weight, pt, 0, dDX, lddx, params ? (float *)workspace : nullptr, vecs, n};
    long long parts = 0;
    if (vecs > 0 && (dDX || params)) {
        const auto run = xt == 0 ? norm_backward_f32 : xt == 1 ? norm_backward_f16 : norm_backward_bf16;
        const tcaspmm_status s = run(p, dim, &parts, st);
        if (s != TCASPMM_OK) return s;
    }
    if (!params) return TCASPMM_OK;
    norm_join<<<dim3(blocks_of(ceil_div(n, 32)), 2), 1024, 0, st>>>((const float *)workspace, parts, n, dweight, dbias, pt);
    return launched("layer_norm_backward launch");
}
