// Group norm with an activation on channels-last tokens, forward and backward (hno_gncl_fwd, hno_gncl_bwd).
//
//   x (B, V, C), group g = C / G neighbouring channels: mean, var over (V, g);  xh = (x - mean) rstd;  u = xh gamma + beta;  y = act(u)
//   du = dy act'(u);  dbeta = sum du;  dgamma = sum du xh;  dx = rstd (du gamma - mean(du gamma) - xh mean(du gamma xh))
//
// Passes over x are what these kernels cost.  A thread owns a few neighbouring channels and walks rows, so a row is read in one piece; the
// sums of a run of rows go to a slab, and one workgroup per group joins the slabs in a fixed order.
// Statistics: no row is special.  Each thread keeps a running mean and sum of squared distances of its rows, re-centred every four rows; the lanes of a run are
// joined around a mean of several of them, the runs in 64 bits.  Neither a channel far from zero nor an outlier in any row (a padded volume's first voxel, a
// spectrum's constant mode) makes large numbers cancel.
// Bound by memory: 2 x 491520 x 64 bf16 (126 MB a tensor), elu: statistics 25 us, result 44, backward sums 51, gradient 62 (5.0, 5.7, 4.9 and 6.1 TB/s, some of it from the
// last-level cache; walking the rows backwards in the second passes, to find more there, changed nothing), joins 6 and 8.  65^3 x 24 fp32 forward 8 + 6 + 13 us.
#include "hno_tokens.h"

#include <type_traits>

namespace hno {

struct GnArgs {
    const void *x, *dy;
    const float *gamma, *beta;
    void *y, *dx;
    float *mr, *slab, *coef, *dgamma, *dbeta;       // mr, coef: (B, G, 2)
    long long V, rows_per;
    int B, C, G, act, runs, cw, chunks;             // cw: channel chunks per workgroup (threads across), chunks: C / W
    float eps;
};

template <typename T, int W>
struct GnVec { float v[W]; };
template <typename T, int W>
__device__ __forceinline__ GnVec<T, W> gn_load(const T *p) {
    GnVec<T, W> r;
    if constexpr (W == 8) {
        const TkFrag<T> f = tk_row(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) r.v[j] = (float)f.v[j];
    } else {
        r.v[0] = tk_up(p[0]);
    }
    return r;
}
template <typename T, int W>
__device__ __forceinline__ void gn_store(T *p, const GnVec<T, W> &r) {
    if constexpr (W == 8) {
        TkFrag<T> f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f.set(j, r.v[j]);
        tk_store8(p, f);
    } else {
        p[0] = tk_down<T>(r.v[0]);
    }
}

// f(activation as a constant): one loop for each activation instead of a branch for each value
template <typename F>
__device__ __forceinline__ void gn_with_act(int act, F f) {
    switch (act) {
        case HNO_ACT_SELU: f(std::integral_constant<int, HNO_ACT_SELU>()); break;
        case HNO_ACT_ELU: f(std::integral_constant<int, HNO_ACT_ELU>()); break;
        case HNO_ACT_RELU: f(std::integral_constant<int, HNO_ACT_RELU>()); break;
        case HNO_ACT_GELU: f(std::integral_constant<int, HNO_ACT_GELU>()); break;
        case HNO_ACT_SILU: f(std::integral_constant<int, HNO_ACT_SILU>()); break;
        default: f(std::integral_constant<int, HNO_ACT_NONE>());
    }
}

// the same, kept as it lies in memory
template <typename T, int W> struct GnRaw { TkFrag<T> f; };
template <typename T> struct GnRaw<T, 1> { T f; };
template <typename T, int W>
__device__ __forceinline__ GnRaw<T, W> gn_raw(const T *p) {
    if constexpr (W == 8) return {tk_row(p)};
    else return {p[0]};
}
template <typename T, int W>
__device__ __forceinline__ float gn_at(const GnRaw<T, W> &r, int j) {
    if constexpr (W == 8) return (float)r.f.v[j];
    else return tk_up(r.f);
}

// sums of the workgroup's rows -> the first two of slab[b][run][ROWS][C].  The lanes that own the same channels meet in LDS; each of the 2 W cw sums is taken by `per` neighbouring
// threads (with one thread a sum, 24 channels left 3 of 256 threads 1360 additions each: 26 us for 65^3 x 24 instead of 8).
template <int W, int ROWS>
__device__ __forceinline__ void gn_block_sums(const GnArgs &a, float (&s1)[W], float (&s2)[W], int nrl, int tid, float *lds) {
    constexpr int S = 2 * W + 1;
#pragma unroll
    for (int j = 0; j < W; ++j) lds[tid * S + j] = s1[j], lds[tid * S + W + j] = s2[j];
    __syncthreads();
    const int nout = 2 * W * a.cw;
    int per = 1;
    while (per < 64 && 2 * per * nout <= 256) per *= 2;
    float *dst = a.slab + ((long long)blockIdx.z * a.runs + blockIdx.x) * ROWS * a.C;
    for (int o0 = 0; o0 < nout; o0 += 256 / per) {
        const int o = o0 + tid / per, sl = tid & (per - 1), ch = o / (2 * W), j = o - ch * 2 * W, c = (blockIdx.y * a.cw + ch) * W;
        const bool on = o < nout && c < a.C;
        float t = 0.f;
        if (on)
            for (int r = sl; r < nrl; r += per) t += lds[(ch + r * a.cw) * S + j];
        for (int k = per >> 1; k; k >>= 1) t += __shfl_xor(t, k);
        if (on && sl == 0) dst[j < W ? c + j : a.C + c + j - W] = t;
    }
}

// per channel and run of rows: a reference value and the sums of x - reference and (x - reference)^2 (three slab rows)
template <typename T, int W>
__global__ __launch_bounds__(256) void gncl_stats_kernel(GnArgs a) {
    __shared__ float lds[256 * (2 * W + 1)];
    __shared__ float refs[256 * W];
    const int tid = threadIdx.x, nrl = 256 / a.cw, rl = tid / a.cw, chunk = blockIdx.y * a.cw + tid - rl * a.cw;
    const long long r0 = (long long)blockIdx.x * a.rows_per, r1 = r0 + a.rows_per < a.V ? r0 + a.rows_per : a.V;
    const bool own = chunk < a.chunks && rl < nrl && r0 + rl < r1;
    float p[W], m[W], q[W], n = 0.f;          // p: the thread's first row; n rows of mean p + m, q: their squared distances from it
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = m[j] = q[j] = 0.f;
    if (own) {
        const T *x = (const T *)a.x + (long long)blockIdx.z * a.V * a.C + chunk * W;
        const GnVec<T, W> first = gn_load<T, W>(x + (r0 + rl) * a.C);
#pragma unroll
        for (int j = 0; j < W; ++j) p[j] = first.v[j];
        // k more rows with deviations d from the mean: mean += sum d / n, q += sum d^2 - (sum d)^2 / n with the new n.  The difference takes at most half of
        // sum d^2; of the first four rows, one of whose d is zero, three quarters.
        const auto rows4 = [&](long long r, auto whole) {
            GnRaw<T, W> v[4];
            bool in[4];
            int k = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                in[i] = whole || r + i * nrl < r1;
                k += in[i];
                v[i] = gn_raw<T, W>(x + (in[i] ? r + i * nrl : r) * a.C);
            }
            n += (float)k;
            const float inv = __builtin_amdgcn_rcpf(n);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float s = 0.f, t = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float d = in[i] ? (gn_at(v[i], j) - p[j]) - m[j] : 0.f;
                    s += d;
                    t = fmaf(d, d, t);
                }
                m[j] = fmaf(s, inv, m[j]);
                q[j] += fmaf(-s * inv, s, t);
            }
        };
        long long r = r0 + rl;
        for (; r + 3 * nrl < r1; r += 4 * nrl) rows4(r, std::true_type());
        if (r < r1) rows4(r, std::false_type());
    }
    // the run's reference: the mean of the means of its first (at most eight) lanes, an outlier's share of it being small
#pragma unroll
    for (int j = 0; j < W; ++j) lds[tid * (W + 1) + j] = p[j] + m[j];
    __syncthreads();
    const int few = (int)min((long long)min(nrl, 8), r1 - r0);
    for (int o = tid; o < W * a.cw; o += 256) {
        const int ch = o / W, j = o - ch * W, c = (blockIdx.y * a.cw + ch) * W + j;
        float t = 0.f;
        for (int l = 0; l < few; ++l) t += lds[(ch + l * a.cw) * (W + 1) + j];
        t /= (float)few;
        refs[o] = t;
        if (c < a.C) a.slab[(((long long)blockIdx.z * a.runs + blockIdx.x) * 3 + 2) * a.C + c] = t;
    }
    __syncthreads();
    float s1[W], s2[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const float d = own ? (p[j] - refs[(tid - rl * a.cw) * W + j]) + m[j] : 0.f;
        s1[j] = n * d;
        s2[j] = fmaf(n * d, d, q[j]);
    }
    gn_block_sums<W, 3>(a, s1, s2, nrl, tid, lds);
}

// joins the runs of a group in 64 bits: with mean_i, M2_i of channel run i of n_i values and any reference r,
//   N (mean - r) = sum n_i (mean_i - r),  M2 = sum M2_i + sum n_i (mean_i - r)^2 - N (mean - r)^2      (r: the first run's reference)
__global__ __launch_bounds__(1024) void gncl_finish_kernel(GnArgs a) {
    __shared__ double sh[2][1024];
    const int tid = threadIdx.x, g = blockIdx.x, b = blockIdx.y, cpg = a.C / a.G;
    const float *slab = a.slab + (long long)b * a.runs * 3 * a.C + g * cpg;
    const double ref = slab[2ll * a.C], inv = 1.0 / (double)a.rows_per, left = (double)(a.V - (a.runs - 1) * a.rows_per), inv_last = 1.0 / left;
    double d1 = 0.0, m2 = 0.0;
#pragma unroll 4
    for (long long i = tid; i < (long long)cpg * a.runs; i += 1024) {
        const int run = (int)(i / cpg), c = (int)(i - (long long)run * cpg);
        const bool last = run == a.runs - 1;
        const float *src = slab + run * 3ll * a.C + c;
        const double n = last ? left : (double)a.rows_per, s1 = src[0], s2 = src[a.C];
        const double mi = s1 * (last ? inv_last : inv), d = (double)src[2ll * a.C] - ref + mi;
        d1 += n * d;
        m2 += s2 - s1 * mi + n * d * d;
    }
    sh[0][tid] = d1, sh[1][tid] = m2;
    for (int o = 512; o; o >>= 1) {
        __syncthreads();
        if (tid < o) sh[0][tid] += sh[0][tid + o], sh[1][tid] += sh[1][tid + o];
    }
    if (tid == 0) {
        const double N = (double)a.V * cpg, d = sh[0][0] / N, var = (sh[1][0] - N * d * d) / N;
        a.mr[2 * (b * a.G + g)] = (float)(ref + d);
        a.mr[2 * (b * a.G + g) + 1] = (float)(1.0 / sqrt((var > 0.0 ? var : (var == var ? 0.0 : var)) + (double)a.eps));
    }
}

template <typename T, int W>
__global__ __launch_bounds__(256) void gncl_apply_kernel(GnArgs a) {
    const int tid = threadIdx.x, nrl = 256 / a.cw, rl = tid / a.cw, chunk = blockIdx.y * a.cw + tid - rl * a.cw, b = blockIdx.z, cpg = a.C / a.G;
    if (chunk >= a.chunks || rl >= nrl) return;
    float mean[W], ga[W], be[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const int c = chunk * W + j, g = c / cpg;
        mean[j] = a.mr[2 * (b * a.G + g)];
        ga[j] = a.mr[2 * (b * a.G + g) + 1] * (a.gamma ? a.gamma[c] : 1.f);
        be[j] = a.beta ? a.beta[c] : 0.f;
    }
    const long long base = (long long)b * a.V * a.C + chunk * W;
    const long long r1 = ((long long)blockIdx.x + 1) * a.rows_per < a.V ? ((long long)blockIdx.x + 1) * a.rows_per : a.V;
    gn_with_act(a.act, [&](auto act) {
#pragma unroll 2
        for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
            GnVec<T, W> v = gn_load<T, W>((const T *)a.x + base + r * a.C);
#pragma unroll
            for (int j = 0; j < W; ++j) v.v[j] = tk_act(fmaf(v.v[j] - mean[j], ga[j], be[j]), act);
            gn_store<T, W>((T *)a.y + base + r * a.C, v);
        }
    });
}

// per channel: sum du and sum du xh over a run of rows
template <typename T, int W>
__global__ __launch_bounds__(256) void gncl_bwd_sums_kernel(GnArgs a) {
    __shared__ float lds[256 * (2 * W + 1)];
    const int tid = threadIdx.x, nrl = 256 / a.cw, rl = tid / a.cw, chunk = blockIdx.y * a.cw + tid - rl * a.cw, b = blockIdx.z, cpg = a.C / a.G;
    float s1[W], s2[W];
#pragma unroll
    for (int j = 0; j < W; ++j) s1[j] = s2[j] = 0.f;
    if (chunk < a.chunks && rl < nrl) {
        float mean[W], rstd[W], ga[W], be[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int c = chunk * W + j, g = c / cpg;
            mean[j] = a.mr[2 * (b * a.G + g)];
            rstd[j] = a.mr[2 * (b * a.G + g) + 1];
            ga[j] = a.gamma ? a.gamma[c] : 1.f;
            be[j] = a.beta ? a.beta[c] : 0.f;
        }
        const long long base = (long long)b * a.V * a.C + chunk * W;
        const long long r1 = ((long long)blockIdx.x + 1) * a.rows_per < a.V ? ((long long)blockIdx.x + 1) * a.rows_per : a.V;
        gn_with_act(a.act, [&](auto act) {
#pragma unroll 2
            for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
                const GnVec<T, W> v = gn_load<T, W>((const T *)a.x + base + r * a.C), d = gn_load<T, W>((const T *)a.dy + base + r * a.C);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float xh = (v.v[j] - mean[j]) * rstd[j], du = d.v[j] * tk_act_grad(fmaf(xh, ga[j], be[j]), act);
                    s1[j] += du;
                    s2[j] = fmaf(du, xh, s2[j]);
                }
            }
        });
    }
    gn_block_sums<W, 2>(a, s1, s2, nrl, tid, lds);
}

// one workgroup per group: dgamma, dbeta of its channels and, per sample, mean(du gamma) and mean(du gamma xh).  `cw` threads across the
// channels, the others across the runs.
__global__ __launch_bounds__(1024) void gncl_bwd_finish_kernel(GnArgs a, int cw) {
    __shared__ float sh[2][1024];
    const int tid = threadIdx.x, cpg = a.C / a.G, g = blockIdx.x, cl = tid & (cw - 1), rl = tid / cw, nrl = 1024 / cw;
    for (int c0 = 0; c0 < cpg; c0 += cw) {
        const int c = g * cpg + c0 + cl;
        const bool on = c0 + cl < cpg;
        float db = 0.f, dg = 0.f;
        for (int b = 0; b < a.B; ++b) {
            float s1 = 0.f, s2 = 0.f;
            const float *src = a.slab + (long long)b * a.runs * 2 * a.C + c;
            if (on)
#pragma unroll 8
                for (int r = rl; r < a.runs; r += nrl) {
                    s1 += src[r * 2ll * a.C];
                    s2 += src[(r * 2ll + 1) * a.C];
                }
            __syncthreads();
            sh[0][tid] = s1, sh[1][tid] = s2;
            for (int o = 512; o >= cw; o >>= 1) {          // across the runs
                __syncthreads();
                if (tid < o) sh[0][tid] += sh[0][tid + o], sh[1][tid] += sh[1][tid + o];
            }
            __syncthreads();
            if (tid < cw) {
                db += sh[0][tid], dg += sh[1][tid];
                const float w = on && a.gamma ? a.gamma[c] : 1.f;
                sh[0][tid] *= w, sh[1][tid] *= w;
            }
            for (int o = cw >> 1; o; o >>= 1) {            // across the channels
                __syncthreads();
                if (tid < o) sh[0][tid] += sh[0][tid + o], sh[1][tid] += sh[1][tid + o];
            }
            if (tid == 0)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float *dst = &a.coef[2 * (b * a.G + g) + k];
                    const float t = c0 ? *dst + sh[k][0] : sh[k][0];
                    *dst = c0 + cw >= cpg ? t / ((float)a.V * (float)cpg) : t;
                }
        }
        if (tid < cw && on) {
            if (a.dbeta) a.dbeta[c] = db;
            if (a.dgamma) a.dgamma[c] = dg;
        }
    }
}

template <typename T, int W>
__global__ __launch_bounds__(256) void gncl_bwd_apply_kernel(GnArgs a) {
    const int tid = threadIdx.x, nrl = 256 / a.cw, rl = tid / a.cw, chunk = blockIdx.y * a.cw + tid - rl * a.cw, b = blockIdx.z, cpg = a.C / a.G;
    if (chunk >= a.chunks || rl >= nrl) return;
    float mean[W], rstd[W], ga[W], be[W], t1[W], t2[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const int c = chunk * W + j, g = c / cpg, k = 2 * (b * a.G + g);
        mean[j] = a.mr[k];
        rstd[j] = a.mr[k + 1];
        ga[j] = a.gamma ? a.gamma[c] : 1.f;
        be[j] = a.beta ? a.beta[c] : 0.f;
        t1[j] = a.coef[k];
        t2[j] = a.coef[k + 1];
    }
    const long long base = (long long)b * a.V * a.C + chunk * W;
    const long long r1 = ((long long)blockIdx.x + 1) * a.rows_per < a.V ? ((long long)blockIdx.x + 1) * a.rows_per : a.V;
    gn_with_act(a.act, [&](auto act) {
#pragma unroll 2
        for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
            GnVec<T, W> v = gn_load<T, W>((const T *)a.x + base + r * a.C);
            const GnVec<T, W> d = gn_load<T, W>((const T *)a.dy + base + r * a.C);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float xh = (v.v[j] - mean[j]) * rstd[j], du = d.v[j] * tk_act_grad(fmaf(xh, ga[j], be[j]), act);
                v.v[j] = rstd[j] * (fmaf(du, ga[j], -t1[j]) - xh * t2[j]);
            }
            gn_store<T, W>((T *)a.dx + base + r * a.C, v);
        }
    });
}

// ------------------------------------------------------------------ small groups: one launch
// A workgroup owns one group of one sample and keeps it in registers: x is read once, the statistics are those of the kept values (mean first, then the
// distances from it and their squares: what the distances add up to corrects the mean, which lost bits if the group's first value is far from it), and the backward
// pass needs no second launch but the sum over samples of dgamma, dbeta.  Threads: chunk (of W channels) x row; a thread keeps gn_keep rows.
// 2 x 960 x 256 bf16 in 32 groups: forward 9.5 us of kernels (in three launches 20), backward 13.8 (31); what is left are the latencies of a launch, a load, two or
// three sums over the workgroup and a store.
constexpr int GN_THREADS = 1024;
template <typename T, int W, bool BWD> constexpr int gn_keep() { return BWD && sizeof(T) == 4 && W == 8 ? 4 : 8; }       // (128 registers a thread)
template <typename T, int W, bool BWD> inline bool gn_small(long long V, int cpg) {
    return cpg % W == 0 && cpg / W <= 64 && V <= (long long)(GN_THREADS / (cpg / W)) * gn_keep<T, W, BWD>();
}
__device__ __forceinline__ float gn_block_sum(float v, float *sh, int tid) {
#pragma unroll
    for (int k = 32; k; k >>= 1) v += __shfl_xor(v, k);
    __syncthreads();
    if ((tid & 63) == 0) sh[tid >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < GN_THREADS / 64; ++k) s += sh[k];
    return s;
}
// two sums for the latency of one
__device__ __forceinline__ void gn_block_sum2(float &v, float &w, float (&sh)[2][GN_THREADS / 64], int tid) {
#pragma unroll
    for (int k = 32; k; k >>= 1) v += __shfl_xor(v, k), w += __shfl_xor(w, k);
    __syncthreads();
    if ((tid & 63) == 0) sh[0][tid >> 6] = v, sh[1][tid >> 6] = w;
    __syncthreads();
    v = w = 0.f;
#pragma unroll
    for (int k = 0; k < GN_THREADS / 64; ++k) v += sh[0][k], w += sh[1][k];
}
template <typename T, int W>
__global__ __launch_bounds__(GN_THREADS) void gncl_small_fwd_kernel(GnArgs a) {
    __shared__ float sh[2][GN_THREADS / 64];
    const int tid = threadIdx.x, g = blockIdx.x, b = blockIdx.y, cpg = a.C / a.G, nch = cpg / W, nr = GN_THREADS / nch, rl = tid / nch, c = g * cpg + (tid - rl * nch) * W;
    constexpr int KEEP = gn_keep<T, W, false>();
    const T *x = (const T *)a.x + (long long)b * a.V * a.C + c;
    const float first = tk_up(((const T *)a.x)[(long long)b * a.V * a.C + g * cpg]), n = (float)a.V * (float)cpg;
    GnRaw<T, W> v[KEEP];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const int r = rl + k * nr;
        const bool in = rl < nr && r < a.V;
        if (in) v[k] = gn_raw<T, W>(x + (long long)r * a.C);
#pragma unroll
        for (int j = 0; j < W; ++j) s += in ? gn_at(v[k], j) - first : 0.f;
    }
    float mean = first + gn_block_sum(s, sh[0], tid) / n, e = 0.f;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const bool in = rl < nr && rl + k * nr < a.V;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float d = in ? gn_at(v[k], j) - mean : 0.f;
            e += d;
            s = fmaf(d, d, s);
        }
    }
    gn_block_sum2(s, e, sh, tid);
    const float var = fmaf(-e / n, e, s) / n, rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    mean += e / n;
    if (tid == 0) a.mr[2 * (b * a.G + g)] = mean, a.mr[2 * (b * a.G + g) + 1] = rstd;
    float ga[W], be[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        ga[j] = rstd * (a.gamma ? a.gamma[c + j] : 1.f);
        be[j] = a.beta ? a.beta[c + j] : 0.f;
    }
    T *y = (T *)a.y + (long long)b * a.V * a.C + c;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const int r = rl + k * nr;
        if (!(rl < nr && r < a.V)) continue;
        GnVec<T, W> u;
#pragma unroll
        for (int j = 0; j < W; ++j) u.v[j] = tk_act(fmaf(gn_at(v[k], j) - mean, ga[j], be[j]), a.act);
        gn_store<T, W>(y + (long long)r * a.C, u);
    }
}
// slab: (B, 2, C), the sums of each sample
template <typename T, int W>
__global__ __launch_bounds__(GN_THREADS) void gncl_small_bwd_kernel(GnArgs a) {
    __shared__ float part[GN_THREADS * (2 * W + 1)];
    __shared__ float tot[2 * 64 * W];
    const int tid = threadIdx.x, g = blockIdx.x, b = blockIdx.y, cpg = a.C / a.G, nch = cpg / W, nr = GN_THREADS / nch, rl = tid / nch, ch = tid - rl * nch, c = g * cpg + ch * W;
    const T *x = (const T *)a.x + (long long)b * a.V * a.C + c, *dy = (const T *)a.dy + (long long)b * a.V * a.C + c;
    const float mean = a.mr[2 * (b * a.G + g)], rstd = a.mr[2 * (b * a.G + g) + 1];
    float ga[W], be[W], s1[W], s2[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        ga[j] = a.gamma ? a.gamma[c + j] : 1.f;
        be[j] = a.beta ? a.beta[c + j] : 0.f;
        s1[j] = s2[j] = 0.f;
    }
    constexpr int KEEP = gn_keep<T, W, true>();
    GnRaw<T, W> v[KEEP], d[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const int r = rl + k * nr;
        if (rl < nr && r < a.V) {
            v[k] = gn_raw<T, W>(x + (long long)r * a.C);
            d[k] = gn_raw<T, W>(dy + (long long)r * a.C);
        }
    }
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (rl < nr && rl + k * nr < a.V)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float xh = (gn_at(v[k], j) - mean) * rstd, du = gn_at(d[k], j) * tk_act_grad(fmaf(xh, ga[j], be[j]), a.act);
                s1[j] += du;
                s2[j] = fmaf(du, xh, s2[j]);
            }
    // per channel: 2 cpg sums over the nr row lanes, each by several threads, then by one
#pragma unroll
    for (int j = 0; j < W; ++j) part[tid * (2 * W + 1) + j] = s1[j], part[tid * (2 * W + 1) + W + j] = s2[j];
    __syncthreads();
    const int nout = 2 * cpg, per = GN_THREADS / nout, o = tid / (per > 0 ? per : 1), sl = tid - o * per;      // (cpg <= 64 W <= 512: per >= 1)
    const int wh = o >= cpg, oc = o - wh * cpg, at = (oc / W) * (2 * W + 1) + wh * W + oc % W;
    float t = 0.f;
    if (o < nout)
        for (int r = sl; r < nr; r += per) t += part[r * nch * (2 * W + 1) + at];
    __syncthreads();
    part[tid] = t;
    __syncthreads();
    if (tid < nout) {
        t = 0.f;
        for (int k = 0; k < per; ++k) t += part[tid * per + k];
        const int cc = g * cpg + (tid < cpg ? tid : tid - cpg);
        if (a.B == 1) {
            if (tid < cpg ? a.dbeta != nullptr : a.dgamma != nullptr) (tid < cpg ? a.dbeta : a.dgamma)[cc] = t;
        } else {
            a.slab[((long long)b * 2 + (tid >= cpg)) * a.C + cc] = t;
        }
        tot[tid] = t * (a.gamma ? a.gamma[cc] : 1.f);
    }
    __syncthreads();
    if (!a.dx) return;
    float t1 = 0.f, t2 = 0.f;
    for (int k = 0; k < cpg; ++k) t1 += tot[k], t2 += tot[cpg + k];
    const float inv = 1.f / ((float)a.V * (float)cpg);
    t1 *= inv, t2 *= inv;
    T *dx = (T *)a.dx + (long long)b * a.V * a.C + c;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const int r = rl + k * nr;
        if (!(rl < nr && r < a.V)) continue;
        GnVec<T, W> u;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float xh = (gn_at(v[k], j) - mean) * rstd, du = gn_at(d[k], j) * tk_act_grad(fmaf(xh, ga[j], be[j]), a.act);
            u.v[j] = rstd * (fmaf(du, ga[j], -t1) - xh * t2);
        }
        gn_store<T, W>(dx + (long long)r * a.C, u);
    }
}
__global__ __launch_bounds__(256) void gncl_params_kernel(GnArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    float db = 0.f, dg = 0.f;
    for (int b = 0; b < a.B; ++b) {
        db += a.slab[(b * 2ll) * a.C + c];
        dg += a.slab[(b * 2ll + 1) * a.C + c];
    }
    if (a.dbeta) a.dbeta[c] = db;
    if (a.dgamma) a.dgamma[c] = dg;
}

}  // namespace hno

using namespace hno;

struct GnPlan {
    int W, cw, chunks, yblocks, runs;
    long long rows_per;
};
static GnPlan gn_plan(int dtype, int B, long long V, int C, bool vec) {
    GnPlan p;
    p.W = vec ? 8 : 1;
    p.chunks = C / p.W;
    p.cw = p.chunks < 256 ? p.chunks : 256;
    p.yblocks = ceil_div(p.chunks, p.cw);
    // (four workgroups a CU: 2 x 491520 x 64 bf16 forward and backward 195 us of kernels; with eight 205, the joins have more runs to read; with two 229, too few
    // loads are on their way)
    const long long nrl = 256 / p.cw, most = 1024 / ((long long)B * p.yblocks) > 1 ? 1024 / ((long long)B * p.yblocks) : 1;
    long long runs = (V + 4 * nrl - 1) / (4 * nrl);            // four rows per thread at least
    if (runs > most) runs = most;
    if (runs < 1) runs = 1;
    p.rows_per = (V + runs - 1) / runs;
    p.runs = (int)((V + p.rows_per - 1) / p.rows_per);
    return p;
}
static int gn_check(const char *what, int dtype, int B, long long V, int C, int G, int act) {
    HNO_REQUIRE(dtype == HNO_F32 || dtype == HNO_BF16, "%s: dtype %d is neither HNO_F32 nor HNO_BF16", what, dtype);
    HNO_REQUIRE(B > 0 && V > 0 && C > 0 && G > 0, "%s: bad size", what);
    HNO_REQUIRE(C % G == 0, "%s: %d channels do not fall into %d groups", what, C, G);
    HNO_REQUIRE(act == HNO_ACT_NONE || act == HNO_ACT_SELU || act == HNO_ACT_ELU || act == HNO_ACT_RELU || act == HNO_ACT_GELU || act == HNO_ACT_SILU,
                "%s: activation %d", what, act);
    if (B > 65535 || C > (1 << 20) || V > (1ll << 40) || (long long)B * G >= 1ll << 30) return fail(HNO_ELIMIT, "%s: a size exceeds the grid", what);
    return HNO_OK;
}
static size_t gn_pad(size_t b) { return (b + 255) / 256 * 256; }
static bool gn_vec(int C, const void *p0, const void *p1, const void *p2) {
    return C % 8 == 0 && ((reinterpret_cast<uintptr_t>(p0) | reinterpret_cast<uintptr_t>(p1) | reinterpret_cast<uintptr_t>(p2)) & 15) == 0;
}
static GnArgs gn_args(const GnPlan &p, int B, long long V, int C, int G, int act) {
    GnArgs a = {};
    a.B = B; a.V = V; a.C = C; a.G = G; a.act = act; a.runs = p.runs; a.rows_per = p.rows_per; a.cw = p.cw; a.chunks = p.chunks;
    return a;
}

#define GN_LAUNCH(KERNEL)                                                                             \
    do {                                                                                              \
        const dim3 grid_(p.runs, p.yblocks, B);                                                       \
        if (p.W == 8) hipLaunchKernelGGL((KERNEL<T, 8>), grid_, dim3(256), 0, s, a);                  \
        else hipLaunchKernelGGL((KERNEL<T, 1>), grid_, dim3(256), 0, s, a);                           \
        HNO_CHECK_LAUNCH();                                                                           \
    } while (0)

template <typename T>
static int gn_forward(const void *x, const float *gamma, const float *beta, void *y, float *mr, void *ws, int B, long long V, int C, int G, float eps, int act,
                      hipStream_t s) {
    const GnPlan p = gn_plan(0, B, V, C, gn_vec(C, x, y, nullptr));
    GnArgs a = gn_args(p, B, V, C, G, act);
    a.x = x; a.gamma = gamma; a.beta = beta; a.y = y; a.mr = mr; a.eps = eps; a.slab = (float *)ws;
    ProfScope _ps(KID_GNCL, s, 2.0 * sizeof(T) * B * V * C);
    if (p.W == 8 && gn_small<T, 8, false>(V, C / G)) {
        hipLaunchKernelGGL((gncl_small_fwd_kernel<T, 8>), dim3(G, B), dim3(GN_THREADS), 0, s, a);
        HNO_CHECK_LAUNCH();
        return HNO_OK;
    }
    if (gn_small<T, 1, false>(V, C / G)) {
        hipLaunchKernelGGL((gncl_small_fwd_kernel<T, 1>), dim3(G, B), dim3(GN_THREADS), 0, s, a);
        HNO_CHECK_LAUNCH();
        return HNO_OK;
    }
    GN_LAUNCH(gncl_stats_kernel);
    hipLaunchKernelGGL(gncl_finish_kernel, dim3(G, B), dim3(1024), 0, s, a);
    HNO_CHECK_LAUNCH();
    GN_LAUNCH(gncl_apply_kernel);
    return HNO_OK;
}
template <typename T>
static int gn_backward(const void *dy, const void *x, const float *gamma, const float *beta, const float *mr, void *dx, float *dgamma, float *dbeta, void *ws,
                       int B, long long V, int C, int G, int act, hipStream_t s) {
    const GnPlan p = gn_plan(0, B, V, C, gn_vec(C, x, dy, dx));
    GnArgs a = gn_args(p, B, V, C, G, act);
    a.x = x; a.dy = dy; a.gamma = gamma; a.beta = beta; a.mr = const_cast<float *>(mr); a.dx = dx; a.dgamma = dgamma; a.dbeta = dbeta;
    a.coef = (float *)ws;
    a.slab = (float *)((char *)ws + gn_pad((size_t)B * G * 2 * sizeof(float)));
    ProfScope _ps(KID_GNCL, s, 3.0 * sizeof(T) * B * V * C);
    const bool s8 = p.W == 8 && gn_small<T, 8, true>(V, C / G);
    if (s8 || gn_small<T, 1, true>(V, C / G)) {
        if (s8) hipLaunchKernelGGL((gncl_small_bwd_kernel<T, 8>), dim3(G, B), dim3(GN_THREADS), 0, s, a);
        else hipLaunchKernelGGL((gncl_small_bwd_kernel<T, 1>), dim3(G, B), dim3(GN_THREADS), 0, s, a);
        HNO_CHECK_LAUNCH();
        if (B > 1 && (dgamma || dbeta)) {
            hipLaunchKernelGGL(gncl_params_kernel, dim3(ceil_div(C, 256)), dim3(256), 0, s, a);
            HNO_CHECK_LAUNCH();
        }
        return HNO_OK;
    }
    GN_LAUNCH(gncl_bwd_sums_kernel);
    int cw = 1;
    while (cw < C / G && cw < 1024) cw *= 2;
    hipLaunchKernelGGL(gncl_bwd_finish_kernel, dim3(G), dim3(1024), 0, s, a, cw);
    HNO_CHECK_LAUNCH();
    if (dx) GN_LAUNCH(gncl_bwd_apply_kernel);
    return HNO_OK;
}

// the larger of the two plans (vector or single channels): which one runs depends on the tensors' alignment
extern "C" size_t hno_gncl_workspace_bytes(int B, long long V, int C, int G) {
    if (gn_check("hno_gncl_workspace_bytes", HNO_F32, B, V, C, G, 0)) return 0;
    const int r0 = gn_plan(0, B, V, C, false).runs, r1 = C % 8 == 0 ? gn_plan(0, B, V, C, true).runs : 0;
    return gn_pad((size_t)B * G * 2 * sizeof(float)) + (size_t)B * (r0 > r1 ? r0 : r1) * 3 * C * sizeof(float);       // (small groups: B x 2 x C)
}
extern "C" int hno_gncl_fwd(int dtype, const void *x, const float *gamma, const float *beta, void *y, float *mean_rstd, void *workspace, size_t workspace_bytes,
                            int B, long long V, int C, int G, float eps, int act, void *stream) {
    if (int rc = gn_check("hno_gncl_fwd", dtype, B, V, C, G, act)) return rc;
    HNO_REQUIRE(x && y && mean_rstd && workspace && eps >= 0.f, "hno_gncl_fwd: bad argument");
    HNO_REQUIRE(workspace_bytes >= hno_gncl_workspace_bytes(B, V, C, G), "hno_gncl_fwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                hno_gncl_workspace_bytes(B, V, C, G));
    if (dtype == HNO_BF16) return gn_forward<tkh>(x, gamma, beta, y, mean_rstd, workspace, B, V, C, G, eps, act, (hipStream_t)stream);
    return gn_forward<float>(x, gamma, beta, y, mean_rstd, workspace, B, V, C, G, eps, act, (hipStream_t)stream);
}
extern "C" int hno_gncl_bwd(int dtype, const void *dy, const void *x, const float *gamma, const float *beta, const float *mean_rstd, void *dx, float *dgamma,
                            float *dbeta, void *workspace, size_t workspace_bytes, int B, long long V, int C, int G, int act, void *stream) {
    if (int rc = gn_check("hno_gncl_bwd", dtype, B, V, C, G, act)) return rc;
    HNO_REQUIRE(dy && x && mean_rstd && workspace && (dx || dgamma || dbeta), "hno_gncl_bwd: bad argument");
    HNO_REQUIRE(workspace_bytes >= hno_gncl_workspace_bytes(B, V, C, G), "hno_gncl_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                hno_gncl_workspace_bytes(B, V, C, G));
    if (dtype == HNO_BF16)
        return gn_backward<tkh>(dy, x, gamma, beta, mean_rstd, dx, dgamma, dbeta, workspace, B, V, C, G, act, (hipStream_t)stream);
    return gn_backward<float>(dy, x, gamma, beta, mean_rstd, dx, dgamma, dbeta, workspace, B, V, C, G, act, (hipStream_t)stream);
}
