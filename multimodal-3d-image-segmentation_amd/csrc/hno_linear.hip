// Matrix product with its epilogue, forward and backward (hno_linear_fwd, hno_linear_bwd).
//
//   z = x W^T + b,  y = act(z) + r                    x (M, K), W (N, K), y (M, N)
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz
//
// One kernel for the three products: C(m, n) = sum_k A(m, k) B(n, k), each operand stored either along k (row reads) or across it
// (transposed reads of the LDS tile: ds_read_b64_tr_b16).  The product is formed as B A^T, so a lane holds four neighbouring columns of
// one output row.  A sum over a long k with few tiles is cut into runs, whose fp32 slabs are added in run order.
#include "hno_tokens.h"

namespace hno {

struct LinArgs {
    const void *A, *B, *bias, *res;
    void *z, *y;
    float *part;
    long long lda, ldb;
    int M, N, K, va, vb, vc, act, bias32, out32, nsplit;
};

constexpr int LN_T = 128;                                   // tile: 128 x 128, four waves of 64 x 64
template <typename T> constexpr int ln_kb() { return sizeof(T) == 2 ? 64 : 32; }

// tile of one operand: `along` k: LN_T rows of KB; across: KB rows of LN_T
template <typename T, bool ACROSS> constexpr int ln_stride() { return (ACROSS ? LN_T : ln_kb<T>()) + tk_pad<T>(); }
template <typename T, bool ACROSS> constexpr int ln_tile() { return (ACROSS ? ln_kb<T>() : LN_T) * ln_stride<T, ACROSS>(); }

template <typename T, bool ACROSS>
__device__ __forceinline__ void ln_stage(T *tile, const T *base, long long ld, int m0, int M, int k0, int K, bool vec, int tid) {
    constexpr int KB = ln_kb<T>(), S = ln_stride<T, ACROSS>(), W = ACROSS ? LN_T : KB, R = ACROSS ? KB : LN_T, CH = W / 8;
    const int row0 = ACROSS ? k0 : m0, rows = ACROSS ? K : M, col0 = ACROSS ? m0 : k0, cols = ACROSS ? M : K;
#pragma unroll
    for (int c = tid; c < R * CH; c += 256) {
        const int row = c / CH, d = (c - row * CH) * 8;
        TkFrag<T> f;
        if (row0 + row < rows) {
            f = tk_load8(base + (long long)(row0 + row) * ld, col0 + d, cols, vec);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f.set(j, 0.f);
        }
        tk_store8(tile + row * S + d, f);
    }
}
template <typename T, bool ACROSS>
__device__ __forceinline__ TkFrag<T> ln_frag(const T *tile, int m0, int kk, int lane) {
    constexpr int S = ln_stride<T, ACROSS>();
    const int k = 16 * kk + 8 * (lane >> 5);
    if constexpr (ACROSS) return tk_col(tile, S, m0, k, k + 4, lane);
    else return tk_row(tile + (m0 + (lane & 31)) * S + k);
}

// the epilogue of four neighbouring columns n .. n + 3 of row m
template <typename T>
__device__ __forceinline__ void ln_finish(const LinArgs &a, int m, int n, float (&x)[4]) {
    const int cnt = a.N - n < 4 ? a.N - n : 4;
    const long long at = (long long)m * a.N + n;
    if (a.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cnt) x[j] += a.bias32 ? ((const float *)a.bias)[n + j] : tk_up(((const T *)a.bias)[n + j]);
    }
    T zs[4];
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.res) {
        if (a.vc) {
            if constexpr (sizeof(T) == 2) {
                const tks4 t = *reinterpret_cast<const tks4 *>((const T *)a.res + at);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = tk_up((tkh)t[j]);
            } else {
                const tkf4 t = *reinterpret_cast<const tkf4 *>((const T *)a.res + at);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = t[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cnt) r[j] = tk_up(((const T *)a.res)[at + j]);
        }
    }
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        zs[j] = tk_down<T>(x[j]);
        y[j] = tk_act(x[j], a.act) + r[j];
    }
    if (a.z) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cnt) ((T *)a.z)[at + j] = zs[j];
    }
    if (a.out32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cnt) ((float *)a.y)[at + j] = y[j];
    } else if (a.vc && sizeof(T) == 2) {
        tks4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (short)tk_down<tkh>(y[j]);
        *reinterpret_cast<tks4 *>((tkh *)a.y + at) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cnt) ((T *)a.y)[at + j] = tk_down<T>(y[j]);
    }
}

template <typename T, bool AX, bool BX>
__global__ __launch_bounds__(256) void linear_kernel(LinArgs a) {
    constexpr int KB = ln_kb<T>();
    __shared__ __attribute__((aligned(16))) T As[ln_tile<T, AX>()];
    __shared__ __attribute__((aligned(16))) T Bs[ln_tile<T, BX>()];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int n0 = blockIdx.x * LN_T, m0 = blockIdx.y * LN_T;
    const int steps = (a.K + KB - 1) / KB, per = (steps + a.nsplit - 1) / a.nsplit;
    const int k1 = ((int)blockIdx.z + 1) * per < steps ? ((int)blockIdx.z + 1) * per : steps;
    tk16 acc[2][2] = {};
    for (int ks = blockIdx.z * per; ks < k1; ++ks) {
        __syncthreads();
        ln_stage<T, AX>(As, (const T *)a.A, a.lda, m0, a.M, ks * KB, a.K, a.va, tid);
        ln_stage<T, BX>(Bs, (const T *)a.B, a.ldb, n0, a.N, ks * KB, a.K, a.vb, tid);
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < KB / 16; ++kk) {
            TkFrag<T> fa[2], fb[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                fa[u] = ln_frag<T, AX>(As, wm + 32 * u, kk, lane);
                fb[u] = ln_frag<T, BX>(Bs, wn + 32 * u, kk, lane);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 2; ++v) acc[u][v] = tk_mma(fb[v], fa[u], acc[u][v]);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int m = m0 + wm + 32 * u + (lane & 31);
        if (m >= a.M) continue;
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = n0 + wn + 32 * v + 8 * q + 4 * h;
                if (n >= a.N) continue;
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = acc[u][v][4 * q + j];
                if (a.nsplit > 1) {
                    float *dst = a.part + ((long long)blockIdx.z * a.M + m) * a.N + n;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n + j < a.N) dst[j] = x[j];
                } else {
                    ln_finish<T>(a, m, n, x);
                }
            }
    }
}

// sum of the runs' slabs, then the epilogue
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(LinArgs a) {
    const int per_row = (a.N + 3) / 4;
    const long long items = (long long)a.M * per_row, slab = (long long)a.M * a.N;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < items; i += (long long)gridDim.x * 256) {
        const int m = (int)(i / per_row), n = 4 * (int)(i - (long long)m * per_row);
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.nsplit; ++s) {
            const float *src = a.part + s * slab + (long long)m * a.N + n;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < a.N) x[j] += src[j];
        }
        ln_finish<T>(a, m, n, x);
    }
}

// dz = dy act'(z) and the column sums of dz: a workgroup owns 64 columns of a run of rows and leaves one slab row per run.
// dz == nullptr: act is none, dz is dy itself and only the sums are wanted.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T *__restrict__ dy, const T *__restrict__ z, T *__restrict__ dz, float *__restrict__ slab,
                                                        int M, int N, int act, int rows_per) {
    __shared__ float red[4][64];
    const int n = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
    const int m0 = blockIdx.y * rows_per, m1 = m0 + rows_per < M ? m0 + rows_per : M;
    float s = 0.f;
    if (n < N)
        for (int m = m0 + w; m < m1; m += 4) {
            const long long at = (long long)m * N + n;
            float g = tk_up(dy[at]);
            if (dz) {
                g *= tk_act_grad(tk_up(z[at]), act);
                dz[at] = tk_down<T>(g);
            }
            s += g;
        }
    if (!slab) return;
    red[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w == 0 && n < N) slab[(long long)blockIdx.y * N + n] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}
template <typename T>
__global__ __launch_bounds__(1024) void linear_db_kernel(const float *__restrict__ slab, int runs, int N, void *db, int db32) {
    __shared__ float red[16][64];
    const int c = threadIdx.x & 63, n = blockIdx.x * 64 + c, w = threadIdx.x >> 6;
    float s = 0.f;
    if (n < N)
        for (int r = w; r < runs; r += 16) s += slab[(long long)r * N + n];
    red[w][c] = s;
    __syncthreads();
    if (w == 0 && n < N) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += red[k][c];
        if (db32) ((float *)db)[n] = t;
        else ((T *)db)[n] = tk_down<T>(t);
    }
}

}  // namespace hno

using namespace hno;

// runs of the contraction: enough workgroups for the chip, no run shorter than four steps
static int ln_splits(int M, int N, int K, int kb) {
    const long long tiles = (long long)ceil_div(M, LN_T) * ceil_div(N, LN_T), steps = ceil_div(K, kb);
    long long n = tiles >= 256 ? 1 : (512 + tiles - 1) / tiles;
    if (n > steps / 4) n = steps / 4;
    if (n > 64) n = 64;
    return n < 1 ? 1 : (int)n;
}
static int ln_runs(int M) { return M <= 64 ? 1 : (ceil_div(M, 64) < 256 ? ceil_div(M, 64) : 256); }
static size_t ln_pad(size_t b) { return (b + 255) / 256 * 256; }
static bool ln_aligned(const void *p, long long ld, int esz) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * esz % 16 == 0; }

template <typename T, bool AX, bool BX>
static int ln_product(LinArgs a, hipStream_t s, int kid) {
    const int esz = sizeof(T);
    // 16-byte reads: the read axis of each operand in whole chunks of 8
    a.va = ln_aligned(a.A, a.lda, esz) && (AX ? a.M : a.K) % 8 == 0;
    a.vb = ln_aligned(a.B, a.ldb, esz) && (BX ? a.N : a.K) % 8 == 0;
    a.vc = a.N % 4 == 0 && ln_aligned(a.y, 0, 1) && ln_aligned(a.res, 0, 1) && !a.out32;
    a.nsplit = ln_splits(a.M, a.N, a.K, ln_kb<T>());
    ProfScope _ps(kid, s, esz * ((double)a.M * a.K + (double)a.N * a.K + (double)a.M * a.N));
    hipLaunchKernelGGL((linear_kernel<T, AX, BX>), dim3(ceil_div(a.N, LN_T), ceil_div(a.M, LN_T), a.nsplit), dim3(256), 0, s, a);
    HNO_CHECK_LAUNCH();
    if (a.nsplit > 1) {
        const long long items = (long long)a.M * ((a.N + 3) / 4), blocks = (items + 255) / 256;
        hipLaunchKernelGGL((linear_join_kernel<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, a);
        HNO_CHECK_LAUNCH();
    }
    return HNO_OK;
}

static int ln_check(const char *what, int dtype, int M, int N, int K, int act) {
    HNO_REQUIRE(dtype == HNO_F32 || dtype == HNO_BF16, "%s: dtype %d is neither HNO_F32 nor HNO_BF16", what, dtype);
    HNO_REQUIRE(M > 0 && N > 0 && K > 0, "%s: bad size", what);
    HNO_REQUIRE(act == HNO_ACT_NONE || act == HNO_ACT_SELU || act == HNO_ACT_ELU || act == HNO_ACT_RELU || act == HNO_ACT_GELU || act == HNO_ACT_SILU,
                "%s: activation %d", what, act);
    if (M > LN_T * 65535ll || N > LN_T * 65535ll || K > LN_T * 65535ll) return fail(HNO_ELIMIT, "%s: a size exceeds the grid", what);
    return HNO_OK;
}
static size_t ln_slab(int M, int N, int K, int kb) {
    const int n = ln_splits(M, N, K, kb);
    return n > 1 ? (size_t)n * M * N * sizeof(float) : 0;
}

extern "C" size_t hno_linear_workspace_bytes(int dtype, int M, int N, int K, int act, int backward) {
    if (ln_check("hno_linear_workspace_bytes", dtype, M, N, K, act)) return 0;
    const int kb = dtype == HNO_BF16 ? ln_kb<tkh>() : ln_kb<float>();
    if (!backward) return ln_slab(M, N, K, kb);
    const size_t dx = ln_slab(M, K, N, kb), dw = ln_slab(N, K, M, kb), dz = act == HNO_ACT_NONE ? 0 : (size_t)M * N * (dtype == HNO_BF16 ? 2 : 4);
    return ln_pad(dz) + ln_pad((size_t)ln_runs(M) * N * sizeof(float)) + (dx > dw ? dx : dw);
}

extern "C" int hno_linear_fwd(int dtype, const void *x, long long ldx, const void *w, const void *bias, int bias_dtype, const void *residual, void *z, void *y,
                              int M, int N, int K, int act, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = ln_check("hno_linear_fwd", dtype, M, N, K, act)) return rc;
    HNO_REQUIRE(x && w && y && ldx >= K, "hno_linear_fwd: bad argument");
    const size_t need = hno_linear_workspace_bytes(dtype, M, N, K, act, 0);
    HNO_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "hno_linear_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    LinArgs a = {};
    a.A = x; a.lda = ldx; a.B = w; a.ldb = K; a.bias = bias; a.bias32 = bias_dtype == HNO_F32; a.res = residual; a.z = z; a.y = y;
    a.M = M; a.N = N; a.K = K; a.act = act; a.part = (float *)workspace;
    if (dtype == HNO_BF16) return ln_product<tkh, false, false>(a, (hipStream_t)stream, KID_LINEAR);
    return ln_product<float, false, false>(a, (hipStream_t)stream, KID_LINEAR);
}

template <typename T>
static int ln_backward(const void *dy, const void *z, const void *x, long long ldx, const void *w, void *dx, void *dw, int dw_dtype, void *db, int db_dtype,
                       int M, int N, int K, int act, char *ws, hipStream_t s) {
    const int runs = ln_runs(M);
    T *dz = act == HNO_ACT_NONE ? nullptr : (T *)ws;
    float *slab = (float *)(ws + ln_pad(dz ? (size_t)M * N * sizeof(T) : 0)), *part = (float *)((char *)slab + ln_pad((size_t)runs * N * sizeof(float)));
    if (dz || db) {
        ProfScope _ps(KID_LINEAR, s, (double)M * N * sizeof(T) * (dz ? 3 : 1));
        hipLaunchKernelGGL((linear_dz_kernel<T>), dim3(ceil_div(N, 64), runs), dim3(256), 0, s, (const T *)dy, (const T *)z, dz, db ? slab : nullptr, M, N, act,
                           ceil_div(M, runs));
        HNO_CHECK_LAUNCH();
        if (db) {
            hipLaunchKernelGGL((linear_db_kernel<T>), dim3(ceil_div(N, 64)), dim3(1024), 0, s, (const float *)slab, runs, N, db, db_dtype == HNO_F32);
            HNO_CHECK_LAUNCH();
        }
    }
    const void *d = dz ? (const void *)dz : dy;
    LinArgs a = {};
    a.part = part;
    if (dx) {
        a.A = d; a.lda = N; a.B = w; a.ldb = K; a.y = dx; a.M = M; a.N = K; a.K = N;
        if (int rc = ln_product<T, false, true>(a, s, KID_LINEAR)) return rc;
    }
    if (dw) {
        a.A = d; a.lda = N; a.B = x; a.ldb = ldx; a.y = dw; a.out32 = sizeof(T) == 2 && dw_dtype == HNO_F32; a.M = N; a.N = K; a.K = M;
        if (int rc = ln_product<T, true, true>(a, s, KID_LINEAR)) return rc;
    }
    return HNO_OK;
}

extern "C" int hno_linear_bwd(int dtype, const void *dy, const void *z, const void *x, long long ldx, const void *w, void *dx, void *dw, int dw_dtype, void *db,
                              int db_dtype, int M, int N, int K, int act, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = ln_check("hno_linear_bwd", dtype, M, N, K, act)) return rc;
    HNO_REQUIRE(dy && (act == HNO_ACT_NONE || z) && (!dx || w) && (!dw || (x && ldx >= K)) && (dx || dw || db), "hno_linear_bwd: bad argument");
    const size_t need = hno_linear_workspace_bytes(dtype, M, N, K, act, 1);
    HNO_REQUIRE(workspace && workspace_bytes >= need, "hno_linear_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (dtype == HNO_BF16) return ln_backward<tkh>(dy, z, x, ldx, w, dx, dw, dw_dtype, db, db_dtype, M, N, K, act, (char *)workspace, (hipStream_t)stream);
    return ln_backward<float>(dy, z, x, ldx, w, dx, dw, dw_dtype, db, db_dtype, M, N, K, act, (char *)workspace, (hipStream_t)stream);
}
