// Group norm with an activation on channels-last tokens, forward and backward (hno_gncl_fwd, hno_gncl_bwd).
//
//   x (B, V, C), group g = C / G neighbouring channels: mean, var over (V, g);  xh = (x - mean) rstd;  u = xh gamma + beta;  y = act(u)
//   du = dy act'(u);  dbeta = sum du;  dgamma = sum du xh;  dx = rstd (du gamma - mean(du gamma) - xh mean(du gamma xh))
//
// Passes over x are what these kernels cost.  A thread owns a few neighbouring channels and walks rows, so a row is read in one piece; the
// sums of a run of rows go to a slab, and one workgroup per group joins the slabs in a fixed order.
// Statistics: each thread sums x - p and (x - p)^2 with p the first row's value of its channel, so a channel far from zero loses nothing; the runs'
// (count, mean, M2) are joined pairwise in 64 bits.
#include "hno_tokens.h"

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

// sums of the workgroup's rows: lanes that own the same channels are added through LDS; slab[b][run][2][C]
template <int W>
__device__ __forceinline__ void gn_block_sums(const GnArgs &a, float (&s1)[W], float (&s2)[W], int chunk, int rl, int nrl, int tid, float *lds) {
#pragma unroll
    for (int j = 0; j < W; ++j) lds[tid * (2 * W + 1) + j] = s1[j], lds[tid * (2 * W + 1) + W + j] = s2[j];
    __syncthreads();
    if (rl != 0 || chunk >= a.chunks) return;
    float *dst = a.slab + ((long long)blockIdx.z * a.runs + blockIdx.x) * 2 * a.C + chunk * W;
#pragma unroll
    for (int j = 0; j < W; ++j) {
        float t1 = 0.f, t2 = 0.f;
        for (int r = 0; r < nrl; ++r) {
            t1 += lds[(tid + r * a.cw) * (2 * W + 1) + j];
            t2 += lds[(tid + r * a.cw) * (2 * W + 1) + W + j];
        }
        dst[j] = t1;
        dst[a.C + j] = t2;
    }
}

template <typename T, int W>
__global__ __launch_bounds__(256) void gncl_stats_kernel(GnArgs a) {
    __shared__ float lds[256 * (2 * W + 1)];
    const int tid = threadIdx.x, nrl = 256 / a.cw, rl = tid / a.cw, chunk = blockIdx.y * a.cw + tid - rl * a.cw;
    float s1[W], s2[W];
#pragma unroll
    for (int j = 0; j < W; ++j) s1[j] = s2[j] = 0.f;
    if (chunk < a.chunks && rl < nrl) {
        const T *x = (const T *)a.x + (long long)blockIdx.z * a.V * a.C + chunk * W;
        const long long r1 = ((long long)blockIdx.x + 1) * a.rows_per < a.V ? ((long long)blockIdx.x + 1) * a.rows_per : a.V;
        const GnVec<T, W> p = gn_load<T, W>(x);
        for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
            const GnVec<T, W> v = gn_load<T, W>(x + r * a.C);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float d = v.v[j] - p.v[j];
                s1[j] += d;
                s2[j] = fmaf(d, d, s2[j]);
            }
        }
    }
    gn_block_sums<W>(a, s1, s2, chunk, rl, nrl, tid, lds);
}

// (count, mean, M2) of two disjoint sets
__device__ __forceinline__ void gn_join(double &n, double &mean, double &m2, double n2, double mean2, double m22) {
    if (n2 == 0.0) return;
    const double t = n + n2, d = mean2 - mean;
    mean += d * n2 / t;
    m2 += m22 + d * d * n * n2 / t;
    n = t;
}
template <typename T>
__global__ __launch_bounds__(256) void gncl_finish_kernel(GnArgs a) {
    __shared__ double sh[3][256];
    const int tid = threadIdx.x, g = blockIdx.x, b = blockIdx.y, cpg = a.C / a.G;
    const T *x = (const T *)a.x + (long long)b * a.V * a.C;
    double n = 0.0, mean = 0.0, m2 = 0.0;
    for (long long i = tid; i < (long long)cpg * a.runs; i += 256) {
        const int run = (int)(i / cpg), c = g * cpg + (int)(i - (long long)run * cpg);
        const long long left = a.V - run * a.rows_per;
        const double cnt = (double)(left < a.rows_per ? left : a.rows_per);
        const float *src = a.slab + ((long long)b * a.runs + run) * 2 * a.C + c;
        const double s1 = src[0], s2 = src[a.C];
        gn_join(n, mean, m2, cnt, (double)tk_up(x[c]) + s1 / cnt, s2 - s1 * s1 / cnt);
    }
    sh[0][tid] = n, sh[1][tid] = mean, sh[2][tid] = m2;
    for (int o = 128; o; o >>= 1) {
        __syncthreads();
        if (tid < o) {
            gn_join(n, mean, m2, sh[0][tid + o], sh[1][tid + o], sh[2][tid + o]);
            sh[0][tid] = n, sh[1][tid] = mean, sh[2][tid] = m2;
        }
    }
    if (tid == 0) {
        const double var = m2 / n;
        a.mr[2 * (b * a.G + g)] = (float)mean;
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
    for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
        GnVec<T, W> v = gn_load<T, W>((const T *)a.x + base + r * a.C);
#pragma unroll
        for (int j = 0; j < W; ++j) v.v[j] = tk_act(fmaf(v.v[j] - mean[j], ga[j], be[j]), a.act);
        gn_store<T, W>((T *)a.y + base + r * a.C, v);
    }
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
        for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
            const GnVec<T, W> v = gn_load<T, W>((const T *)a.x + base + r * a.C), d = gn_load<T, W>((const T *)a.dy + base + r * a.C);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float xh = (v.v[j] - mean[j]) * rstd[j], du = d.v[j] * tk_act_grad(fmaf(xh, ga[j], be[j]), a.act);
                s1[j] += du;
                s2[j] = fmaf(du, xh, s2[j]);
            }
        }
    }
    gn_block_sums<W>(a, s1, s2, chunk, rl, nrl, tid, lds);
}

// one workgroup per group: dgamma, dbeta of its channels and, per sample, mean(du gamma) and mean(du gamma xh).  `cw` threads across the
// channels, the others across the runs.
__global__ __launch_bounds__(256) void gncl_bwd_finish_kernel(GnArgs a, int cw) {
    __shared__ float sh[2][256];
    __shared__ float tot[2][256];
    const int tid = threadIdx.x, cpg = a.C / a.G, g = blockIdx.x, cl = tid % cw, rl = tid / cw, nrl = 256 / cw;
    for (int c0 = 0; c0 < cpg; c0 += cw) {
        const int c = g * cpg + c0 + cl;
        const bool on = c0 + cl < cpg;
        float db = 0.f, dg = 0.f;
        for (int b = 0; b < a.B; ++b) {
            float s1 = 0.f, s2 = 0.f;
            if (on && rl < nrl)
                for (int r = rl; r < a.runs; r += nrl) {
                    const float *src = a.slab + ((long long)b * a.runs + r) * 2 * a.C + c;
                    s1 += src[0];
                    s2 += src[a.C];
                }
            __syncthreads();
            sh[0][tid] = s1, sh[1][tid] = s2;
            __syncthreads();
            if (tid < cw) {
                s1 = s2 = 0.f;
                for (int r = 0; r < nrl; ++r) s1 += sh[0][r * cw + tid], s2 += sh[1][r * cw + tid];
                db += s1, dg += s2;
                const float w = on ? (a.gamma ? a.gamma[c] : 1.f) : 0.f;
                tot[0][tid] = w * s1, tot[1][tid] = w * s2;
            }
            __syncthreads();
            if (tid < 2) {
                float t = 0.f;
                for (int k = 0; k < cw; ++k) t += tot[tid][k];
                float *dst = &a.coef[2 * (b * a.G + g) + tid];
                t = c0 ? *dst + t : t;
                *dst = c0 + cw >= cpg ? t / ((float)a.V * (float)cpg) : t;
            }
        }
        if (tid < cw && on) {
            if (a.dbeta) a.dbeta[c] = db;
            if (a.dgamma) a.dgamma[c] = dg;
        }
        __syncthreads();
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
    for (long long r = blockIdx.x * a.rows_per + rl; r < r1; r += nrl) {
        GnVec<T, W> v = gn_load<T, W>((const T *)a.x + base + r * a.C);
        const GnVec<T, W> d = gn_load<T, W>((const T *)a.dy + base + r * a.C);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float xh = (v.v[j] - mean[j]) * rstd[j], du = d.v[j] * tk_act_grad(fmaf(xh, ga[j], be[j]), a.act);
            v.v[j] = rstd[j] * (fmaf(du, ga[j], -t1[j]) - xh * t2[j]);
        }
        gn_store<T, W>((T *)a.dx + base + r * a.C, v);
    }
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
    const long long nrl = 256 / p.cw, most = 2048 / ((long long)B * p.yblocks) > 1 ? 2048 / ((long long)B * p.yblocks) : 1;
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
    if (B > 65535 || C > (1 << 20) || V > (1ll << 40)) return fail(HNO_ELIMIT, "%s: a size exceeds the grid", what);
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
    GN_LAUNCH(gncl_stats_kernel);
    hipLaunchKernelGGL((gncl_finish_kernel<T>), dim3(G, B), dim3(256), 0, s, a);
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
    GN_LAUNCH(gncl_bwd_sums_kernel);
    int cw = 1;
    while (cw < C / G && cw < 256) cw *= 2;
    hipLaunchKernelGGL(gncl_bwd_finish_kernel, dim3(G), dim3(256), 0, s, a, cw);
    HNO_CHECK_LAUNCH();
    if (dx) GN_LAUNCH(gncl_bwd_apply_kernel);
    return HNO_OK;
}

// the larger of the two plans (vector or single channels): which one runs depends on the tensors' alignment
extern "C" size_t hno_gncl_workspace_bytes(int B, long long V, int C, int G) {
    if (gn_check("hno_gncl_workspace_bytes", HNO_F32, B, V, C, G, 0)) return 0;
    const int r0 = gn_plan(0, B, V, C, false).runs, r1 = C % 8 == 0 ? gn_plan(0, B, V, C, true).runs : 0;
    return gn_pad((size_t)B * G * 2 * sizeof(float)) + (size_t)B * (r0 > r1 ? r0 : r1) * 2 * C * sizeof(float);
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
