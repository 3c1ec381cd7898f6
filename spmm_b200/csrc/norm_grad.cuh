// The backward kernels of layer norm and their launch, instantiated by the type of X in norm_grad_*.cu.
#pragma once

#include "norm.cuh"

namespace tca {
namespace {

template <typename T, typename G, int VEC, int NCH, int LANES, int THREADS>  // LANES as in norm_rows_fwd
__global__ void __launch_bounds__(THREADS) norm_rows_bwd(const NormGradParams p, int lanes)
{
    constexpr bool BLOCK = THREADS != 256;
    constexpr bool KEEP = VEC * NCH <= 8 || THREADS == 512;
    __shared__ float s[2][2][32];
    extern __shared__ float sum[];  // !BLOCK: a block's partial gradients, added warp by warp
    if (LANES) lanes = LANES;
    const int tpr = BLOCK ? (int)blockDim.x : lanes;
    const int t = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1));
    const int per = BLOCK ? 1 : 256 / lanes;
    const long long first = (long long)blockIdx.x * per + (BLOCK ? 0 : (int)threadIdx.x / lanes);
    const long long step = (long long)gridDim.x * per;
    const int n = (int)p.n;
    const float inv = 1.0f / (float)n;
    float w[KEEP ? VEC * NCH : 1], dw[VEC * NCH], db[VEC * NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = (c * tpr + t) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[c * VEC + e] = db[c * VEC + e] = 0.0f;
        if (KEEP && i < n) load_params<VEC>(p.w, p.pt, p.pvec, i, 1.0f, w + c * VEC);
    }
    Pack<T, VEC> x[NCH], nx[NCH];
    Pack<G, VEC> g[NCH], ng[NCH];
    float mean, rstd, nmean, nrstd;
    auto fetch = [&](long long row, Pack<T, VEC> (&tx)[NCH], Pack<G, VEC> (&tg)[NCH], float &m, float &r) {
        const bool in = row < p.vecs;
        m = in ? __ldg(p.mean + row) : 0.0f;
        r = in ? __ldg(p.rstd + row) : 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int i = (c * tpr + t) * VEC;
            if (in && i < n) {
                tx[c].load((const T *)p.X + row * p.ldx + i);
                tg[c].load((const G *)p.dY + row * p.lddy + i);
            } else {
                tx[c].zero();
                tg[c].zero();
            }
        }
    };
    fetch(first, x, g, mean, rstd);
    const long long turns = (p.vecs - (long long)blockIdx.x * per + step - 1) / step;
    for (long long k = 0; k < turns; ++k) {
        const long long row = first + k * step;
        fetch(row + step, nx, ng, nmean, nrstd);
        float a[2] = {0.0f, 0.0f};
        const bool in = row < p.vecs;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int i = (c * tpr + t) * VEC;
            if (in && i < n) {
                float ww[VEC];
                if (!KEEP) load_params<VEC>(p.w, p.pt, p.pvec, i, 1.0f, ww);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float dy = g[c].get(e), gx = dy * ((x[c].get(e) - mean) * rstd), we = KEEP ? w[c * VEC + e] : ww[e];
                    a[0] = fmaf(dy, we, a[0]);
                    a[1] = fmaf(gx, we, a[1]);
                    dw[c * VEC + e] += gx;
                    db[c * VEC + e] += dy;
                }
            }
        }
        if (p.dX) {
            row_sum<BLOCK>(a, lanes, s[k & 1]);
            const float c1 = a[0] * inv, k2 = rstd * (a[1] * inv);  // dx = rstd (g w - c1 - (x - mean) k2)
            if (in) {
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    const int i = (c * tpr + t) * VEC;
                    if (i < n) {
                        float d[VEC], ww[VEC];
                        if (!KEEP) load_params<VEC>(p.w, p.pt, p.pvec, i, 1.0f, ww);
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            d[e] = rstd * fmaf(g[c].get(e), KEEP ? w[c * VEC + e] : ww[e], -fmaf(x[c].get(e) - mean, k2, c1));
                        store_pack<VEC>((T *)p.dX + row * p.lddx + i, d);
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            x[c] = nx[c];
            g[c] = ng[c];
        }
        mean = nmean;
        rstd = nrstd;
    }
    if (!p.part) return;
    float *pw = p.part + (long long)blockIdx.x * p.n, *pb = pw + (long long)gridDim.x * p.n;
    if constexpr (BLOCK) {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = (c * tpr + t) * VEC + e;
                if (i < n) {
                    pw[i] = dw[c * VEC + e];
                    pb[i] = db[c * VEC + e];
                }
            }
    } else {
        // The groups of `lanes` threads add up in turn: within a warp by shuffles, then the warps one after another.
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (o >= lanes) {
#pragma unroll
                for (int j = 0; j < VEC * NCH; ++j) {
                    dw[j] += __shfl_xor_sync(~0u, dw[j], o);
                    db[j] += __shfl_xor_sync(~0u, db[j], o);
                }
            }
        const int width = lanes * VEC * NCH;
        for (int k = 0; k < (int)(blockDim.x >> 5); ++k) {
            if ((int)(threadIdx.x >> 5) == k && (int)(threadIdx.x & 31) < lanes) {
#pragma unroll
                for (int c = 0; c < NCH; ++c)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int i = (c * lanes + t) * VEC + e;
                        sum[i] = (k ? sum[i] : 0.0f) + dw[c * VEC + e];
                        sum[width + i] = (k ? sum[width + i] : 0.0f) + db[c * VEC + e];
                    }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            pw[i] = sum[i];
            pb[i] = sum[width + i];
        }
    }
}

template <typename T, typename G>
__global__ void __launch_bounds__(STRIP_THREADS) norm_cols_bwd(const NormGradParams p, const Strip q, int vec)
{
    constexpr int VEC = 16 / (int)(sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G));
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float s[2][STRIP_WARPS][STRIP_MAX];
    __shared__ float sums[2][STRIP_MAX];
    __shared__ float fin[2][STRIP_MAX];
    __shared__ float stat[2][STRIP_MAX];  // the columns' mean and rstd
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int width = q.lpr * VEC, at = (threadIdx.x & (q.lpr - 1)) * VEC;
    const long long strip = blockIdx.x / ranks, strips = gridDim.x / ranks, c0 = strip * width;
    const long long r0 = min(p.n, (long long)rank * q.per_block);
    const int rows = (int)(min(p.n, r0 + q.per_block) - r0);
    const int row = threadIdx.x >> q.shift, step = STRIP_THREADS >> q.shift;
    T *const xs = (T *)smem;
    G *const gs = (G *)(smem + ((size_t)q.per_block * width * sizeof(T) + 15) / 16 * 16);  // its vectors' alignment
    float *const ws = (float *)((unsigned char *)gs + ((size_t)q.per_block * width * sizeof(G) + 15) / 16 * 16);  // the rows' weight
    load_strip<T, VEC>(xs, (const T *)p.X, p.ldx, r0, rows, c0, p.vecs, width, q, vec);
    load_strip<G, VEC>(gs, (const G *)p.dY, p.lddy, r0, rows, c0, p.vecs, width, q, vec);
    for (int r = threadIdx.x; r < rows; r += STRIP_THREADS) ws[r] = p.w ? load_as(p.w, p.pt, r0 + r) : 1.0f;
    if ((int)threadIdx.x < width) {
        const bool in = c0 + threadIdx.x < p.vecs;
        stat[0][threadIdx.x] = in ? __ldg(p.mean + c0 + threadIdx.x) : 0.0f;
        stat[1][threadIdx.x] = in ? __ldg(p.rstd + c0 + threadIdx.x) : 0.0f;
    }
    copy_async_wait();
    __syncthreads();
    float mean[VEC], rstd[VEC], v[2][VEC] = {};
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        mean[e] = stat[0][at + e];
        rstd[e] = stat[1][at + e];
    }
    // Columns past the end hold zeros in both arrays and in mean and rstd: they add nothing.
#pragma unroll 2
    for (int first = 0; first < rows; first += step) {  // the same number of turns for all threads of a warp
        const int r = first + row;
        float a = 0.0f, d = 0.0f;
        if (r < rows) {
            const float w = ws[r];
            float x[VEC], g[VEC];
            load_shared<T, VEC>(xs + r * width + at, x);
            load_shared<G, VEC>(gs + r * width + at, g);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float gx = g[e] * ((x[e] - mean[e]) * rstd[e]);
                v[0][e] = fmaf(g[e], w, v[0][e]);
                v[1][e] = fmaf(gx, w, v[1][e]);
                a += gx;
                d += g[e];
            }
        }
        if (p.part) {
            for (int o = q.lpr >> 1; o; o >>= 1) {
                a += __shfl_xor_sync(~0u, a, o);
                d += __shfl_xor_sync(~0u, d, o);
            }
            if (at == 0 && r < rows) {
                p.part[strip * p.n + r0 + r] = a;
                p.part[(strips + strip) * p.n + r0 + r] = d;
            }
        }
    }
    if (!p.dX) return;
    strip_sum(v, q.lpr, s, sums);
    if (ranks > 1) cluster.sync();
    for (int j = threadIdx.x; j < 2 * width; j += STRIP_THREADS) {
        const int k = j / width, c = j - k * width;
        float part[8], t = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) part[i] = i < ranks ? cluster.map_shared_rank(&sums[0][0], i)[k * STRIP_MAX + c] : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += part[i];
        fin[k][c] = t / (float)p.n;
    }
    __syncthreads();
    if (ranks > 1) cluster.barrier_arrive();  // this block has read the others' sums
    if (vec) {
        if (c0 + at < p.vecs) {
            // dx = rstd (g w - c1 - xh c2),  xh c2 = (x - mean) k2,  k2 = rstd c2
            float k1[VEC], k2[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                k1[e] = fin[0][at + e];
                k2[e] = rstd[e] * fin[1][at + e];
            }
            T *out = (T *)p.dX + (r0 + row) * p.lddx + c0 + at;
            const long long down = step * p.lddx;
#pragma unroll 2
            for (int r = row; r < rows; r += step, out += down) {
                const float w = ws[r];
                float x[VEC], g[VEC];
                load_shared<T, VEC>(xs + r * width + at, x);
                load_shared<G, VEC>(gs + r * width + at, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[e] = rstd[e] * fmaf(g[e], w, -fmaf(x[e] - mean[e], k2[e], k1[e]));
                store_pack<VEC>(out, x);
            }
        }
    } else {
        const int c = threadIdx.x & (width - 1), per = STRIP_THREADS / width;
        if (c0 + c < p.vecs) {
            const float m = stat[0][c], rs = stat[1][c], k1 = fin[0][c], k2 = rs * fin[1][c];
            T *out = (T *)p.dX + (r0 + threadIdx.x / width) * p.lddx + c0 + c;
            const long long down = per * p.lddx;
#pragma unroll 4
            for (int r = threadIdx.x / width; r < rows; r += per, out += down)
                *out = from_float<T>(rs * fmaf(to_float(gs[r * width + c]), ws[r], -fmaf(to_float(xs[r * width + c]) - m, k2, k1)));
        }
    }
    if (ranks > 1) cluster.barrier_wait();
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_long_bwd(const NormGradParams p, long long sv, long long si, long long gv, long long gi,
                                                      long long dv, long long di)
{
    __shared__ float s[32];
    for (long long v = blockIdx.x; v < p.vecs; v += gridDim.x) {
        const T *x = (const T *)p.X + v * sv;
        const float mean = p.mean[v], rstd = p.rstd[v];
        float a = 0.0f, c = 0.0f;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float g = load_as(p.dY, p.dyt, v * gv + i * gi) * (p.w ? load_as(p.w, p.pt, i) : 1.0f);
            a += g;
            c += g * ((to_float(x[i * si]) - mean) * rstd);
        }
        a = block_sum(a, s) / (float)p.n;
        c = block_sum(c, s) / (float)p.n;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float g = load_as(p.dY, p.dyt, v * gv + i * gi) * (p.w ? load_as(p.w, p.pt, i) : 1.0f);
            const float xh = (to_float(x[i * si]) - mean) * rstd;
            ((T *)p.dX)[v * dv + i * di] = from_float<T>(rstd * (g - a - xh * c));
        }
    }
}

// Partial weight and bias gradients of rows too long for norm_rows_bwd: a thread per feature, a block row per part.
template <typename T>
__global__ void __launch_bounds__(256) norm_long_rows_wgrad(const NormGradParams p)
{
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= p.n) return;
    float a = 0.0f, c = 0.0f;
    for (long long v = blockIdx.y; v < p.vecs; v += gridDim.y) {
        const float dy = load_as(p.dY, p.dyt, v * p.lddy + i);
        a += dy * ((to_float(((const T *)p.X)[v * p.ldx + i]) - p.mean[v]) * p.rstd[v]);
        c += dy;
    }
    p.part[blockIdx.y * p.n + i] = a;
    p.part[(gridDim.y + blockIdx.y) * p.n + i] = c;
}

// The same of columns too long for norm_cols_bwd: a block per feature, whose values lie side by side.
template <typename T>
__global__ void __launch_bounds__(256) norm_long_cols_wgrad(const NormGradParams p)
{
    __shared__ float s[8];
    for (long long i = blockIdx.x; i < p.n; i += gridDim.x) {
        float a = 0.0f, c = 0.0f;
        for (long long v = threadIdx.x; v < p.vecs; v += blockDim.x) {
            const float dy = load_as(p.dY, p.dyt, i * p.lddy + v);
            a += dy * ((to_float(((const T *)p.X)[i * p.ldx + v]) - p.mean[v]) * p.rstd[v]);
            c += dy;
        }
        a = block_sum(a, s);
        c = block_sum(c, s);
        if (threadIdx.x == 0) {
            p.part[i] = a;
            p.part[p.n + i] = c;
        }
    }
}

template <typename T, typename G, int VEC>
tcaspmm_status backward(const NormGradParams &p, int dim, long long *parts, cudaStream_t st)
{
    const int sms = sm_count();
    if (dim == 1) {
        const RowPlan r = plan_rows(p.n, VEC, BWD_MOST, 1024);
        if (r.nch) {
            // Blocks an SM holds, at most ROW_PARTS: their count is the number of partial gradients.
            const int fit = !r.lanes ? std::min(ROW_PARTS, std::max(1, 512 / r.threads)) : r.nch * VEC > 8 ? 1 : r.nch * VEC > 4 ? 2 : ROW_PARTS;
            const long long grid = std::min(ceil_div(p.vecs, r.lanes ? 256 / r.lanes : 1), (long long)fit * sms);
            *parts = grid;
            return with_chunks<BWD_MOST / VEC>(r.nch, [&](auto nch) {
                constexpr int N = nch.value;
                const size_t shared = r.lanes ? sizeof(float) * 2 * r.lanes * VEC * N : 0;
                if (r.lanes == 32) {
                    norm_rows_bwd<T, G, VEC, N, 32, 256><<<(unsigned)grid, 256, shared, st>>>(p, 32);
                    return launched("layer_norm_backward launch");
                }
                if constexpr (N == 1) {  // a part of a warp: one chunk a thread
                    if (r.lanes) {
                        norm_rows_bwd<T, G, VEC, N, 0, 256><<<(unsigned)grid, 256, shared, st>>>(p, r.lanes);
                        return launched("layer_norm_backward launch");
                    }
                }
                if constexpr (N * VEC * 4 >= BWD_MOST) {  // a block: a quarter of the most, or more
                    if (!r.lanes && r.threads <= 512) {
                        norm_rows_bwd<T, G, VEC, N, 0, 512><<<(unsigned)grid, r.threads, 0, st>>>(p, 32);
                        return launched("layer_norm_backward launch");
                    }
                }
                if constexpr (N * VEC == BWD_MOST) {  // more than 512 threads: the most
                    if (!r.lanes) {
                        norm_rows_bwd<T, G, VEC, N, 0, 1024><<<(unsigned)grid, r.threads, 0, st>>>(p, 32);
                        return launched("layer_norm_backward launch");
                    }
                }
                return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: no kernel for rows of %lld", p.n);
            });
        }
    } else {
        constexpr int WIDE = sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G);
        const StripPlan q = plan_strips(p.n, p.vecs, 16 / WIDE, WIDE, sizeof(T) + sizeof(G), 4, 64, sms);
        static std::atomic<unsigned long long> done{0};
        if (q.ranks && q.strips * q.ranks <= INT_MAX) {
            *parts = q.strips;
            return launch_cluster(norm_cols_bwd<T, G>, q, done, st, p, q.q, (int)(VEC > 1));
        }
    }
    if (p.dX)
        norm_long_bwd<T><<<blocks_of(p.vecs), 1024, 0, st>>>(p, dim ? p.ldx : 1, dim ? 1 : p.ldx, dim ? p.lddy : 1, dim ? 1 : p.lddy,
                                                             dim ? p.lddx : 1, dim ? 1 : p.lddx);
    *parts = 1;
    if (p.part && dim == 1) {
        *parts = std::min<long long>(p.vecs, LONG_PARTS);
        norm_long_rows_wgrad<T><<<dim3(blocks_of(ceil_div(p.n, 256)), (unsigned)*parts), 256, 0, st>>>(p);
    } else if (p.part) {
        norm_long_cols_wgrad<T><<<blocks_of(p.n), 256, 0, st>>>(p);
    }
    return launched("layer_norm_backward launch");
}

}  // namespace

// dX and the partial weight gradients; *parts: how many there are.
template <typename T>
tcaspmm_status norm_backward(NormGradParams p, int dim, long long *parts, cudaStream_t st)
{
    const long long cols = dim == 1 ? p.n : p.vecs;
    const int xt = std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 1 : 2;
    return with_type(p.dyt, [&](auto u) {
        using G = decltype(u);
        constexpr int VEC = 16 / (int)(sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G));
        p.pvec = aligned(p.w, 0, p.pt, VEC);
        if (cols % VEC == 0 && aligned(p.X, p.ldx, xt, VEC) && aligned(p.dY, p.lddy, p.dyt, VEC) && aligned(p.dX, p.lddx, xt, VEC))
            return backward<T, G, VEC>(p, dim, parts, st);
        return backward<T, G, 1>(p, dim, parts, st);
    });
}

}  // namespace tca
