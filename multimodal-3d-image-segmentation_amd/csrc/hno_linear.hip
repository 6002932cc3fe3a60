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
    int M, N, K, act, bias32, out32, nsplit, across;          // across: 1: A is stored across k, 2: B is
    // beside dW: db (db_n) from the slab of column sums, one row a run
    const float *db_slab;
    void *db;
    int db_runs, db_n, db32, db_blocks;
};

// Tiles of the result (TM x TN), contraction elements a step (KB) and the part of one wave (WM x WN).  With 64 x 64 per wave the LDS reads of a step
// take as long as its matrix instructions, with 128 x 64 three quarters.
//   LnBig: large results; LnMid: small ones (more tiles, two workgroups a CU); LnF32: three planes per operand
struct LnBig { static constexpr int TM = 256, TN = 256, KB = 64, WM = 128, WN = 64; };
struct LnMid { static constexpr int TM = 128, TN = 128, KB = 64, WM = 64, WN = 64; };
struct LnF32 { static constexpr int TM = 128, TN = 128, KB = 32, WM = 64, WN = 64; };
template <typename C> constexpr int ln_waves() { return C::TM / C::WM * (C::TN / C::WN); }

// Where 8 elements (chunk c of row r) of an operand's LDS tile stand.  Along k: TILE rows of KB; 16 consecutive rows at one chunk touch all banks.
// Across: KB rows of TILE; 4 consecutive rows at four neighbouring chunks touch all banks (the transposed reads).
template <int TILE, int KB, bool ACROSS>
__device__ __forceinline__ int ln_at(int r, int c) {
    if constexpr (ACROSS) return r * TILE + (c ^ ((r & 3) << 2)) * 8;
    else if constexpr (KB == 64) return r * KB + (c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3))) * 8;
    else return r * KB + (c ^ ((r >> 2) & 3)) * 8;
}

// A workgroup's share of one operand's tile: thread t moves the 8-element slots t, t + threads, ...
template <typename T, int TILE, int KB, int NT, bool ACROSS, bool DMA>
struct LnStage {
    static constexpr int CH = (ACROSS ? TILE : KB) / 8, N = TILE * KB / 8 / NT, PLANE = TILE * KB;
    static constexpr int NR = DMA ? 1 : N;
    TkFrag<T> r[NR];
    unsigned off[DMA ? N : 1];           // DMA: byte offset of each slot's source from the tile's corner
    const T *base;
    long long ld;
    int rows, cols, row0, col0;          // of the stored matrix, and the tile's corner (the corner along k moves)
    __device__ __forceinline__ void init(const void *p, long long ld_, int m0, int M, int K, int tid) {
        base = (const T *)p, ld = ld_;
        rows = ACROSS ? K : M, cols = ACROSS ? M : K, row0 = ACROSS ? 0 : m0, col0 = ACROSS ? m0 : 0;
        if constexpr (DMA)
#pragma unroll
            for (int i = 0; i < N; ++i) off[i] = offset(row(i, tid), source(i, tid) * 8, ACROSS ? KB : rows - row0, ACROSS ? cols - col0 : KB);
    }
    __device__ __forceinline__ static int row(int i, int tid) { return (tid + NT * i) / CH; }
    __device__ __forceinline__ static int chunk(int i, int tid) { return (tid + NT * i) % CH; }
    // DMA (16-byte aligned rows, whole chunks): the chunk whose place the slot is
    __device__ __forceinline__ static int source(int i, int tid) { return (ln_at<TILE, KB, ACROSS>(row(i, tid), chunk(i, tid)) / 8) % CH; }
    // beyond the `nr` rows or `nc` columns left of the matrix: any element of it (settle() clears what must not count)
    __device__ __forceinline__ unsigned offset(int rr, int cc, int nr, int nc) const { return (unsigned)(min(rr, nr - 1) * (int)ld + (cc < nc ? cc : 0)) * 2; }
    // slots i0 ... i1 - 1 (DMA; the last, partial step goes whole with the first of them)
    __device__ __forceinline__ void fetch(tkh *tile, int k0, int tid, int i0 = 0, int i1 = N) {
        const int ra = ACROSS ? k0 : row0, ca = ACROSS ? col0 : k0;
        const T *src = base + (long long)ra * ld + ca;
        const bool whole = ra + (ACROSS ? KB : TILE) <= rows && ca + (ACROSS ? TILE : KB) <= cols;
        if constexpr (DMA) {
            typedef __attribute__((address_space(3))) tkh *ldsp;
            const unsigned dst = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(ldsp)tile + (tid >> 6) * 1024);
            if (k0 + KB <= (ACROSS ? rows : cols)) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i >= i0 && i < i1) tk_dma16(src, off[i], dst + i * NT * 16);
            } else if (i0 == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) tk_dma16(src, offset(row(i, tid), source(i, tid) * 8, rows - ra, cols - ca), dst + i * NT * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int rr = row(i, tid), cc = chunk(i, tid) * 8;
                if (whole || (ra + rr < rows && ca + cc + 8 <= cols)) {
                    __builtin_memcpy(&r[i], src + rr * ld + cc, sizeof(T) * 8);          // any alignment
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) r[i].set(j, ra + rr < rows && ca + cc + j < cols ? tk_up(src[rr * ld + cc + j]) : 0.f);
                }
            }
        }
    }
    __device__ __forceinline__ void settle(tkh *tile, int k0, int K, int tid) {
        if constexpr (DMA) {
            if (k0 + KB > K)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (k0 + (ACROSS ? row(i, tid) : source(i, tid) * 8) >= K) *reinterpret_cast<tku4 *>(tile + (tid + NT * i) * 8) = tku4{0, 0, 0, 0};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                tkh *p = tile + ln_at<TILE, KB, ACROSS>(row(i, tid), chunk(i, tid));
                const TkOp<T> o = tk_op(r[i]);
#pragma unroll
                for (int t = 0; t < tk_planes<T>(); ++t) tk_store8(p + t * PLANE, o.p[t]);
            }
        }
    }
};
template <int TILE, int KB, bool ACROSS>
__device__ __forceinline__ TkFrag<tkh> ln_frag(const tkh *tile, int m0, int kk, int lane) {
    if constexpr (ACROSS) {
        typedef __attribute__((address_space(3))) tks4 *lds4;
        const int r = 16 * kk + 8 * (lane >> 5) + ((lane & 15) >> 2), d = m0 + (lane & 16) + 4 * (lane & 3);
        const tks4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(tile + ln_at<TILE, KB, true>(r, d >> 3) + (d & 7)));
        const tks4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(tile + ln_at<TILE, KB, true>(r + 4, d >> 3) + (d & 7)));
        return {__builtin_bit_cast(tkb8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7))};
    } else {
        return tk_row(tile + ln_at<TILE, KB, false>(m0 + (lane & 31), 2 * kk + (lane >> 5)));
    }
}

// 8 neighbouring values of a row, `cnt` of them inside it; any alignment
template <typename T>
__device__ __forceinline__ TkFrag<T> ln_raw8(const T *p, int cnt) {
    TkFrag<T> f;
    if (cnt >= 8) {
        __builtin_memcpy(&f, p, 8 * sizeof(T));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f.set(j, j < cnt ? tk_up(p[j]) : 0.f);
    }
    return f;
}
template <typename T>
__device__ __forceinline__ void ln_get8(const T *p, int cnt, float (&x)[8]) {
    const TkFrag<T> f = ln_raw8(p, cnt);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)f.v[j];
}
template <typename T>
__device__ __forceinline__ void ln_put8(T *p, int cnt, const float (&x)[8]) {
    if (cnt >= 8) {
        TkFrag<T> f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f.set(j, x[j]);
        __builtin_memcpy(p, &f, 8 * sizeof(T));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < cnt) p[j] = tk_down<T>(x[j]);
    }
}
// fp32: a NaN of columns n .. n + 7 of row m may come from an infinity, whose lower bf16 terms are none: that product once more, in fp32 from the operands.
// It ends at a true NaN; finite results pay a comparison.
__device__ __forceinline__ void ln_infinite(const LinArgs &a, int m, int n, float (&x)[8]) {
    const float none = (x[0] + x[1]) + (x[2] + x[3]) + ((x[4] + x[5]) + (x[6] + x[7]));
    if (none == none) return;
    const float *pa = (const float *)a.A + m * (a.across & 1 ? 1 : a.lda), *pb = (const float *)a.B;
    const long long sa = a.across & 1 ? a.lda : 1, sb = a.across & 2 ? a.ldb : 1, sn = a.across & 2 ? 1 : a.ldb;
    float s[8] = {};
    bool open = true;
#pragma unroll 1
    for (int k = 0; k < a.K && open; ++k) {
        const float v = pa[k * sa];
        open = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = fmaf(v, pb[k * sb + min(n + j, a.N - 1) * sn], s[j]);
            open |= x[j] != x[j] && s[j] == s[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] == x[j] ? x[j] : s[j];
}
// the epilogue of columns n .. n + 7 of row m; r: the residual's values, loaded before
template <typename T, int ACT>
__device__ __forceinline__ void ln_finish(const LinArgs &a, int m, int n, float (&x)[8], const TkFrag<T> &r) {
    const int cnt = a.N - n;
    const long long at = (long long)m * a.N + n;
    if constexpr (sizeof(T) == 4) ln_infinite(a, m, n, x);
    if (a.bias) {
        float t[8];
        if (a.bias32) ln_get8((const float *)a.bias + n, cnt, t);
        else ln_get8((const T *)a.bias + n, cnt, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += t[j];
    }
    if (ACT != HNO_ACT_NONE && a.z) ln_put8((T *)a.z + at, cnt, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = tk_act(x[j], ACT);
    if (a.res)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += (float)r.v[j];
    if (a.out32) ln_put8((float *)a.y + at, cnt, x);
    else ln_put8((T *)a.y + at, cnt, x);
}

// DMA: two LDS buffers, the next step's tiles on their way while this one is multiplied.  Else the next step's tiles wait in registers: one buffer.
// Bound by the matrix pipes: 8192 x 8192 x 2048 bf16, calls back to back, 250 us = 1100 TFLOP/s (the library's product 230), with residual 267, with gelu 272, with bias,
// gelu and residual 300 (LnMid: 330) -- the epilogue of a tile waits for its products, one workgroup a CU.  The first dozen calls of a process take 273, 326 and
// 349 (bare, gelu, everything).  fp32 (six bf16 products each): 2000 x 512 x 512 27 us.
template <typename T, bool AX, bool BX, typename C, bool DMA, int ACT>
__global__ __launch_bounds__(64 * ln_waves<C>(), 2) void linear_kernel(LinArgs a) {
    constexpr int TM = C::TM, TN = C::TN, KB = C::KB, P = tk_planes<T>(), WM = C::WM, WN = C::WN, NT = 64 * ln_waves<C>(), NB = DMA ? 2 : 1;
    constexpr int PA = TM * KB, PB = TN * KB, BUF = P * (PA + PB);      // LDS: A's buffers, then B's
    constexpr int ES = WN + 4, EP = 2 * ln_waves<C>() * 32 * ES;                  // (epilogue: 32 rows of floats a wave)
    __shared__ __attribute__((aligned(16))) tkh smem[EP > NB * BUF ? EP : NB * BUF];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, wm = (wave % (TM / WM)) * WM, wn = (wave / (TM / WM)) * WN;
    // every XCD takes one run of the list of tiles; neighbours in a run share rows (bands of 4 tile rows, column by column)
    const int tm = (a.M + TM - 1) / TM, tn = (a.N + TN - 1) / TN, each = gridDim.x >> 3, more = gridDim.x & 7, xcd = blockIdx.x & 7;
    int at = xcd * each + min(xcd, more) + (blockIdx.x >> 3);
    const int run = at / (tm * tn);
    at -= run * tm * tn;
    const int band = at / (4 * tn), bm = min(4, tm - 4 * band), m0 = (4 * band + (at - band * 4 * tn) % bm) * TM, n0 = ((at - band * 4 * tn) / bm) * TN;
    const int steps = (a.K + KB - 1) / KB, per = (steps + a.nsplit - 1) / a.nsplit, k0 = run * per, k1 = min(k0 + per, steps);
    LnStage<T, TM, KB, NT, AX, DMA> sa;
    LnStage<T, TN, KB, NT, BX, DMA> sb;
    sa.init(a.A, a.lda, m0, a.M, a.K, tid);
    sb.init(a.B, a.ldb, n0, a.N, a.K, tid);
    const auto fetch = [&](int ks, int buf) {
        sa.fetch(smem + buf * P * PA, ks * KB, tid);
        sb.fetch(smem + (NB * PA + buf * PB) * P, ks * KB, tid);
    };
    const auto settle = [&](int ks, int buf) {
        sa.settle(smem + buf * P * PA, ks * KB, a.K, tid);
        sb.settle(smem + (NB * PA + buf * PB) * P, ks * KB, a.K, tid);
    };
    // fragments of chunk kk; two sets where registers allow, so that they are read one chunk ahead of their products
    constexpr int FB = P == 1 ? 2 : 1, KC = KB / 16;
    TkOp<T> fa[FB][WM / 32], fb[FB][WN / 32];
    const auto read = [&](int buf, int kk) {
        const tkh *As = smem + buf * P * PA, *Bs = smem + (NB * PA + buf * PB) * P;
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int v = 0; v < WN / 32; ++v) fb[kk % FB][v].p[p] = ln_frag<TN, KB, BX>(Bs + p * PB, wn + 32 * v, kk, lane);
#pragma unroll
            for (int u = 0; u < WM / 32; ++u) fa[kk % FB][u].p[p] = ln_frag<TM, KB, AX>(As + p * PA, wm + 32 * u, kk, lane);
        }
    };
    tk16 acc[WM / 32][WN / 32] = {};
    const auto multiply = [&](int kk, auto between) {          // between(u): what is issued behind row u of the products
#pragma unroll
        for (int u = 0; u < WM / 32; ++u) {
#pragma unroll
            for (int v = 0; v < WN / 32; ++v) acc[u][v] = tk_mma(fb[kk % FB][v], fa[kk % FB][u], acc[u][v]);
            between(u);
        }
    };
    const auto nothing = [](int) {};
    if constexpr (DMA) {
        // one barrier a step, before its last chunk, whose fragments every wave has by then: behind it the next step's tiles are whole, this step's buffer
        // is free for the step after, and the next step's first fragments are read beside the last chunk's products
        static_assert(NB == 2 && FB == 2 && KC % 2 == 0, "two buffers, an even number of chunks");
        // the DMA of a step's tiles is issued in pieces between products: those of A beside the last chunk, those of B beside the first of the next step
        constexpr int U = WM / 32;
        static_assert(sa.N % U == 0 && sb.N % U == 0, "whole pieces");
        const auto fetch_a = [&](int ks, int buf, int u) { sa.fetch(smem + buf * P * PA, ks * KB, tid, u * (sa.N / U), (u + 1) * (sa.N / U)); };
        const auto fetch_b = [&](int ks, int buf, int u) { sb.fetch(smem + (NB * PA + buf * PB) * P, ks * KB, tid, u * (sb.N / U), (u + 1) * (sb.N / U)); };
        const auto step = [&](int ks, int buf) {
            const bool next = ks + 1 < k1, after = ks + 2 < k1;
            read(buf, 1);
            multiply(0, [&](int u) { if (next) fetch_b(ks + 1, buf ^ 1, u); });
#pragma unroll
            for (int kk = 1; kk + 1 < KC; ++kk) {
                read(buf, kk + 1);
                multiply(kk, nothing);
            }
            if (next) {
                dma_wait<0>();
                settle(ks + 1, buf ^ 1);
                __syncthreads();
                read(buf ^ 1, 0);
            }
            multiply(KC - 1, [&](int u) { if (after) fetch_a(ks + 2, buf, u); });
        };
        if (k0 < k1) {
            fetch(k0, 0);
            if (k0 + 1 < k1)
#pragma unroll
                for (int u = 0; u < U; ++u) fetch_a(k0 + 1, 1, u);
            dma_wait<0>();
            settle(k0, 0);
            __syncthreads();
            read(0, 0);
        }
        for (int ks = k0; ks < k1; ks += 2) {          // (the buffers by name: their addresses are then constants)
            step(ks, 0);
            if (ks + 1 < k1) step(ks + 1, 1);
        }
    } else {
        if (k0 < k1) fetch(k0, 0);
        for (int ks = k0; ks < k1; ++ks) {
            __syncthreads();
            settle(ks, 0);
            __syncthreads();
            if (ks + 1 < k1) fetch(ks + 1, 0);
            if (FB == 2) read(0, 0);
#pragma unroll
            for (int kk = 0; kk < KC; ++kk) {
                if (FB == 1) read(0, kk);
                else if (kk + 1 < KC) read(0, kk + 1);
                multiply(kk, nothing);
            }
        }
    }
    // the results change places in LDS, 32 rows of a wave at a time (its own part: no barrier inside), so that memory is read and written in runs of 128 bytes
    constexpr int PASS = 32 * WN / 8 / 64;
    TkFrag<T> r[WM / 32][PASS];                           // (the residual's loads are all on their way by then)
    if (a.res && a.nsplit == 1)
#pragma unroll
        for (int u = 0; u < WM / 32; ++u)
#pragma unroll
            for (int e = 0; e < PASS; ++e) {
                const int i = lane + 64 * e, m = m0 + wm + 32 * u + i / (WN / 8), n = n0 + wn + (i % (WN / 8)) * 8;
                if (m < a.M && n < a.N) r[u][e] = ln_raw8((const T *)a.res + (long long)m * a.N + n, a.N - n);
            }
    __syncthreads();
    float *ep = reinterpret_cast<float *>(smem) + wave * 32 * ES;
#pragma unroll
    for (int u = 0; u < WM / 32; ++u) {
#pragma unroll
        for (int v = 0; v < WN / 32; ++v)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<tkf4 *>(ep + (lane & 31) * ES + 32 * v + 8 * q + 4 * h) =
                    tkf4{acc[u][v][4 * q], acc[u][v][4 * q + 1], acc[u][v][4 * q + 2], acc[u][v][4 * q + 3]};
#pragma unroll
        for (int e = 0; e < PASS; ++e) {
            const int i = lane + 64 * e, c = (i % (WN / 8)) * 8, m = m0 + wm + 32 * u + i / (WN / 8), n = n0 + wn + c;
            const TkFrag<float> f = tk_row(ep + (i / (WN / 8)) * ES + c);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = f.v[j];
            if (m < a.M && n < a.N) {
                if (a.nsplit > 1) ln_put8(a.part + ((long long)run * a.M + m) * a.N + n, a.N - n, x);
                else ln_finish<T, ACT>(a, m, n, x, r[u][e]);
            }
        }
    }
}

// db of 64 columns: the slab's rows are shared out among the waves
template <typename T, int WAVES>
__device__ __forceinline__ void ln_db(const LinArgs &a, int block) {
    __shared__ float red[WAVES][64];
    const int c = threadIdx.x & 63, n = block * 64 + c, w = threadIdx.x >> 6;
    float s = 0.f;
    if (n < a.db_n)
#pragma unroll 16
        for (int r = w; r < a.db_runs; r += WAVES) s += a.db_slab[(long long)r * a.db_n + n];
    red[w][c] = s;
    __syncthreads();
    if (w == 0 && n < a.db_n) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) t += red[k][c];
        if (a.db32) ((float *)a.db)[n] = t;
        else ((T *)a.db)[n] = tk_down<T>(t);
    }
}
template <typename T>
__global__ __launch_bounds__(1024) void linear_db_kernel(LinArgs a) {
    ln_db<T, 16>(a, blockIdx.x);
}

// sum of the runs' slabs, then the epilogue; the last workgroups take db (a launch less, and 2 us of the 8.5 that both took for 3920 x 1536 x 384 bf16)
template <typename T, int ACT>
__global__ __launch_bounds__(256) void linear_join_kernel(LinArgs a) {
    const int blocks = gridDim.x - a.db_blocks;
    if ((int)blockIdx.x >= blocks) return ln_db<T, 4>(a, blockIdx.x - blocks);
    const int per_row = (a.N + 7) / 8;
    const long long items = (long long)a.M * per_row, slab = (long long)a.M * a.N;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < items; i += (long long)blocks * 256) {
        const int m = (int)(i / per_row), n = 8 * (int)(i - (long long)m * per_row);
        const float *src = a.part + (long long)m * a.N + n;
        float x[8] = {}, t[8];
        TkFrag<T> r = {};
        if (a.res) r = ln_raw8((const T *)a.res + (long long)m * a.N + n, a.N - n);
#pragma unroll 8
        for (int s = 0; s < a.nsplit; ++s) {
            ln_get8(src + s * slab, a.N - n, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] += t[j];
        }
        ln_finish<T, ACT>(a, m, n, x, r);
    }
}

// Up to four rows: bound by reading the weight once, so no tiles.  A workgroup owns two columns, its lanes walk the contraction 8 elements at a time, every
// product and sum in fp32; the lanes' sums meet in shuffles, the waves' in LDS; one launch.  4 x 2048 x 2048: bf16 5.7 us (tiles in 32 runs 10.3), fp32 8.3; bf16 4 x 8192 x 16384:
// 45 us = 6.0 TB/s, the weight partly from the last-level cache; 4 x 16384 x 8192 60 us =
// 4.5 TB/s (72), one row 43 us = 6.2 TB/s (72, the weight partly from the last-level cache).  Eight rows are quicker in tiles (8 x 8192 x 2048: 12.0 us, 30.8 here: every
// workgroup reads all of x).
constexpr int LN_ROWS = 4, LN_COLS = 2;
__device__ __forceinline__ float ln_dot8(const TkFrag<tkh> &x, const TkFrag<tkh> &w, float s) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 8; j += 2) s = __builtin_amdgcn_fdot2_f32_bf16(b2{x.v[j], x.v[j + 1]}, b2{w.v[j], w.v[j + 1]}, s, false);
    return s;
}
__device__ __forceinline__ float ln_dot8(const TkFrag<float> &x, const TkFrag<float> &w, float s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(x.v[j], w.v[j], s);
    return s;
}
template <typename T, int MR>
__global__ __launch_bounds__(256) void linear_rows_kernel(LinArgs a) {
    __shared__ float part[4][MR * LN_COLS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n0 = blockIdx.x * LN_COLS;
    const T *x = (const T *)a.A, *w = (const T *)a.B;
    constexpr int V = MR * LN_COLS;
    float acc[V] = {};
#pragma unroll 2
    for (int k = 8 * tid; k < a.K; k += 8 * 256) {
        const int cnt = a.K - k;
        TkFrag<T> fw[LN_COLS], fx[MR];
#pragma unroll
        for (int c = 0; c < LN_COLS; ++c) fw[c] = ln_raw8(w + (long long)min(n0 + c, a.N - 1) * a.ldb + k, cnt);
#pragma unroll
        for (int m = 0; m < MR; ++m) fx[m] = ln_raw8(x + min(m, a.M - 1) * a.lda + k, cnt);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = ln_dot8(fx[i / LN_COLS], fw[i % LN_COLS], acc[i]);
    }
    // in each exchange a lane hands over the half of its sums that its partner keeps
    int step = 32;
#pragma unroll
    for (int h = V / 2; h; h >>= 1, step >>= 1)
#pragma unroll
        for (int i = 0; i < h; ++i) {
            const bool up = lane & step;
            acc[i] = (up ? acc[i + h] : acc[i]) + __shfl_xor(up ? acc[i] : acc[i + h], step);
        }
    const int left = 2 * step;                          // lanes that hold the same sum
    for (; step; step >>= 1) acc[0] += __shfl_xor(acc[0], step);
    if ((lane & (left - 1)) == 0) part[wave][lane / left] = acc[0];
    __syncthreads();
    const int m = tid / LN_COLS, n = n0 + tid % LN_COLS;
    if (m >= a.M || n >= a.N) return;
    const long long at = (long long)m * a.N + n;
    float z = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    if (a.bias) z += a.bias32 ? ((const float *)a.bias)[n] : tk_up(((const T *)a.bias)[n]);
    if (a.z && a.act != HNO_ACT_NONE) ((T *)a.z)[at] = tk_down<T>(z);
    float y = tk_act(z, a.act);
    if (a.res) y += tk_up(((const T *)a.res)[at]);
    ((T *)a.y)[at] = tk_down<T>(y);
}

// dz = dy act'(z) and the column sums of dz.  dz is rounded to the operator's type, being an operand of two products (db adds it up before that); z was kept in that
// type too: half the memory, for an error of the slope below dz's own rounding where |z| is of order one.
// A workgroup owns 256 columns (32 lanes of 8) of a run of rows and leaves one slab row per run; single columns a lane took 16 us for 3920 x 1536 bf16 instead of 11.
// dz == nullptr: act is none, dz is dy itself and only the sums are wanted.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T *__restrict__ dy, const T *__restrict__ z, T *__restrict__ dz, float *__restrict__ slab,
                                                        int M, int N, int rows_per) {
    __shared__ float red[8][32 * 9];
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockIdx.x * 256 + 8 * c, cnt = N - n;
    const int m0 = blockIdx.y * rows_per, m1 = min(m0 + rows_per, M);
    float s[8] = {};
    if (cnt > 0)
#pragma unroll 2
        for (int m = m0 + w; m < m1; m += 8) {
            const long long at = (long long)m * N + n;
            float g[8];
            ln_get8(dy + at, cnt, g);
            if constexpr (ACT != HNO_ACT_NONE) {
                float t[8];
                ln_get8(z + at, cnt, t);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] *= tk_act_grad(t[j], ACT);
                ln_put8(dz + at, cnt, g);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += g[j];
        }
    if (!slab) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[w][9 * c + j] = s[j];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x, at = 9 * (threadIdx.x >> 3) + (threadIdx.x & 7);
    if (col >= N) return;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][at];
    slab[(long long)blockIdx.y * N + col] = t;
}

}  // namespace hno

using namespace hno;

// Tile, and runs of the contraction.  LnBig (8192 x 8192 x 8192 bf16: 1238 TFLOP/s, LnMid 1034) where its tiles fill most of the 256 CUs by themselves and DMA can
// feed it.  Else 128 x 128 tiles, whose contraction is cut into n runs where that is expected to be quicker: a step takes a workgroup 0.65 us (fp32: 2.5) while
// there are places for all (two a CU), the slabs cost 2.5 us for the second launch, 0.12 us each and 0.65 us per megabyte.  Measured with these:
// 3920 x 384 x 1536 bf16 n = 1: 17.2 us (2: 22.5, 4: 24.1), 1536 x 384 x 3920 n = 5: 22.9 (1: 55, 12: 25), 300 x 300 x 4000 n = 8: 13.8 (1: 36, 24: 17.9),
// fp32 771 x 387 x 3001 n = 16: 32.5 (1: 240, 8: 41), 3001 x 387 x 771 n = 5: 32.1 (1: 66, 12: 48), 4096 x 1024 x 256 n = 1: 21.1 (2: 32.8).
struct LnPlan {
    bool big;
    int nsplit;
    long long blocks;
};
static LnPlan ln_plan(int M, int N, int K, bool f32, bool dma) {
    LnPlan p;
    long long tiles = (long long)ceil_div(M, LnBig::TM) * ceil_div(N, LnBig::TN);
    p.big = tiles >= 192 && !f32 && dma;
    p.nsplit = 1;
    if (!p.big) {
        tiles = (long long)ceil_div(M, 128) * ceil_div(N, 128);
        const int steps = ceil_div(K, f32 ? LnF32::KB : LnMid::KB);
        const double step_us = f32 ? 2.5 : 0.65, slab_us = 0.65e-6 * 4.0 * M * N;
        double best = 0.0;
        for (int n = 1; n <= 64 && n <= steps && (n == 1 || tiles * n <= 512); ++n) {
            const double cost = ceil_div(steps, n) * step_us + (n > 1 ? 2.5 + n * (0.12 + slab_us) : 0.0);
            if (n == 1 || cost < best) best = cost, p.nsplit = n;
        }
    }
    p.blocks = tiles * p.nsplit;
    return p;
}
static int ln_runs(int M) { return ceil_div(M, 32) < 256 ? ceil_div(M, 32) : 256; }          // runs of rows of dz: 4 rows a thread at least
static size_t ln_pad(size_t b) { return (b + 255) / 256 * 256; }
static bool ln_aligned(const void *p, long long ld, int esz) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * esz % 16 == 0; }

template <typename T>
static int ln_bias(const LinArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((linear_db_kernel<T>), dim3(ceil_div(a.db_n, 64)), dim3(1024), 0, s, a);
    HNO_CHECK_LAUNCH();
    return HNO_OK;
}
template <typename T, bool AX, bool BX, int ACT>
static int ln_product(LinArgs a, hipStream_t s) {
    const int esz = sizeof(T);
    // DMA: whole 16-byte chunks along the stored axis of each operand, and offsets within a tile in 32 bits
    const bool dma = esz == 2 && ln_aligned(a.A, a.lda, esz) && (AX ? a.M : a.K) % 8 == 0 && ln_aligned(a.B, a.ldb, esz) && (BX ? a.N : a.K) % 8 == 0 &&
                     a.lda < (1 << 22) && a.ldb < (1 << 22);
    const LnPlan p = ln_plan(a.M, a.N, a.K, sizeof(T) == 4, dma);
    if (p.blocks >= 1ll << 23) return fail(HNO_ELIMIT, "hno_linear: %lld tiles exceed the grid", p.blocks);          // (of 2^32 threads)
    a.nsplit = p.nsplit;
    a.across = AX + 2 * BX;
    ProfScope _ps(KID_LINEAR, s, esz * ((double)a.M * a.K + (double)a.N * a.K + (double)a.M * a.N));
    const dim3 grid((unsigned)p.blocks);
    if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((linear_kernel<T, AX, BX, LnF32, false, ACT>), grid, dim3(64 * ln_waves<LnF32>()), 0, s, a);
    else if (p.big) hipLaunchKernelGGL((linear_kernel<T, AX, BX, LnBig, true, ACT>), grid, dim3(64 * ln_waves<LnBig>()), 0, s, a);
    else if (dma) hipLaunchKernelGGL((linear_kernel<T, AX, BX, LnMid, true, ACT>), grid, dim3(64 * ln_waves<LnMid>()), 0, s, a);
    else hipLaunchKernelGGL((linear_kernel<T, AX, BX, LnMid, false, ACT>), grid, dim3(64 * ln_waves<LnMid>()), 0, s, a);
    HNO_CHECK_LAUNCH();
    if (a.nsplit > 1) {
        const long long items = (long long)a.M * ((a.N + 7) / 8), blocks = (items + 255) / 256;
        if (a.db) a.db_blocks = ceil_div(a.db_n, 64);
        hipLaunchKernelGGL((linear_join_kernel<T, ACT>), dim3((unsigned)(blocks < 4096 ? blocks : 4096) + a.db_blocks), dim3(256), 0, s, a);
        HNO_CHECK_LAUNCH();
        return HNO_OK;
    }
    return a.db ? ln_bias<T>(a, s) : HNO_OK;
}

static int ln_check(const char *what, int dtype, int M, int N, int K, int act) {
    HNO_REQUIRE(dtype == HNO_F32 || dtype == HNO_BF16, "%s: dtype %d is neither HNO_F32 nor HNO_BF16", what, dtype);
    HNO_REQUIRE(M > 0 && N > 0 && K > 0, "%s: bad size", what);
    HNO_REQUIRE(act == HNO_ACT_NONE || act == HNO_ACT_SELU || act == HNO_ACT_ELU || act == HNO_ACT_RELU || act == HNO_ACT_GELU || act == HNO_ACT_SILU,
                "%s: activation %d", what, act);
    if (M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) return fail(HNO_ELIMIT, "%s: a size exceeds 2^30", what);
    return HNO_OK;
}
// a tensor beside the operator's own: its type or fp32 (a kernel that took another one for its own would write past its end)
static bool ln_type(const void *t, int dtype, int own) { return !t || dtype == HNO_F32 || dtype == own; }
static size_t ln_slab(int M, int N, int K, bool f32) {
    const int n = ln_plan(M, N, K, f32, false).nsplit;          // (where LnBig is taken, one)
    return n > 1 ? (size_t)n * M * N * sizeof(float) : 0;
}

extern "C" size_t hno_linear_workspace_bytes(int dtype, int M, int N, int K, int act, int backward) {
    if (ln_check("hno_linear_workspace_bytes", dtype, M, N, K, act)) return 0;
    const bool f32 = dtype == HNO_F32;
    if (!backward) return M <= LN_ROWS ? 0 : ln_slab(M, N, K, f32);
    const size_t dx = ln_slab(M, K, N, f32), dw = ln_slab(N, K, M, f32), dz = act == HNO_ACT_NONE ? 0 : (size_t)M * N * (dtype == HNO_BF16 ? 2 : 4);
    return ln_pad(dz) + ln_pad((size_t)ln_runs(M) * N * sizeof(float)) + (dx > dw ? dx : dw);
}

template <typename T>
static int ln_rows(const LinArgs &a, hipStream_t s) {
    ProfScope _ps(KID_LINEAR, s, sizeof(T) * ((double)a.M * a.K + (double)a.N * a.K + (double)a.M * a.N));
    const dim3 grid(ceil_div(a.N, LN_COLS));
    if (grid.x >= 1u << 24) return fail(HNO_ELIMIT, "hno_linear: %d columns exceed the grid", a.N);
    if (a.M == 1) hipLaunchKernelGGL((linear_rows_kernel<T, 1>), grid, dim3(256), 0, s, a);
    else if (a.M == 2) hipLaunchKernelGGL((linear_rows_kernel<T, 2>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((linear_rows_kernel<T, 4>), grid, dim3(256), 0, s, a);
    HNO_CHECK_LAUNCH();
    return HNO_OK;
}
template <typename T>
static int ln_forward(const LinArgs &a, hipStream_t s) {
    if (a.M <= LN_ROWS) return ln_rows<T>(a, s);
    switch (a.act) {
        case HNO_ACT_SELU: return ln_product<T, false, false, HNO_ACT_SELU>(a, s);
        case HNO_ACT_ELU: return ln_product<T, false, false, HNO_ACT_ELU>(a, s);
        case HNO_ACT_RELU: return ln_product<T, false, false, HNO_ACT_RELU>(a, s);
        case HNO_ACT_GELU: return ln_product<T, false, false, HNO_ACT_GELU>(a, s);
        case HNO_ACT_SILU: return ln_product<T, false, false, HNO_ACT_SILU>(a, s);
        default: return ln_product<T, false, false, HNO_ACT_NONE>(a, s);
    }
}

extern "C" int hno_linear_fwd(int dtype, const void *x, long long ldx, const void *w, const void *bias, int bias_dtype, const void *residual, void *z, void *y,
                              int M, int N, int K, int act, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = ln_check("hno_linear_fwd", dtype, M, N, K, act)) return rc;
    HNO_REQUIRE(x && w && y && ldx >= K, "hno_linear_fwd: bad argument");
    HNO_REQUIRE(ln_type(bias, bias_dtype, dtype), "hno_linear_fwd: bias type %d beside type %d", bias_dtype, dtype);
    const size_t need = hno_linear_workspace_bytes(dtype, M, N, K, act, 0);
    HNO_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "hno_linear_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    LinArgs a = {};
    a.A = x; a.lda = ldx; a.B = w; a.ldb = K; a.bias = bias; a.bias32 = bias_dtype == HNO_F32; a.res = residual; a.z = z; a.y = y;
    a.M = M; a.N = N; a.K = K; a.act = act; a.part = (float *)workspace;
    return dtype == HNO_BF16 ? ln_forward<tkh>(a, (hipStream_t)stream) : ln_forward<float>(a, (hipStream_t)stream);
}

template <typename T>
static int ln_backward(const void *dy, const void *z, const void *x, long long ldx, const void *w, void *dx, void *dw, int dw_dtype, void *db, int db_dtype,
                       int M, int N, int K, int act, char *ws, hipStream_t s) {
    const int runs = ln_runs(M);
    T *dz = act == HNO_ACT_NONE ? nullptr : (T *)ws;
    float *slab = (float *)(ws + ln_pad(dz ? (size_t)M * N * sizeof(T) : 0)), *part = (float *)((char *)slab + ln_pad((size_t)runs * N * sizeof(float)));
    if (dz || db) {
        ProfScope _ps(KID_LINEAR, s, (double)M * N * sizeof(T) * (dz ? 3 : 1));
        const dim3 grid(ceil_div(N, 256), runs);
        const int per = ceil_div(M, runs);
#define LN_DZ(ACT) hipLaunchKernelGGL((linear_dz_kernel<T, ACT>), grid, dim3(256), 0, s, (const T *)dy, (const T *)z, dz, db ? slab : nullptr, M, N, per)
        switch (act) {
            case HNO_ACT_SELU: LN_DZ(HNO_ACT_SELU); break;
            case HNO_ACT_ELU: LN_DZ(HNO_ACT_ELU); break;
            case HNO_ACT_RELU: LN_DZ(HNO_ACT_RELU); break;
            case HNO_ACT_GELU: LN_DZ(HNO_ACT_GELU); break;
            case HNO_ACT_SILU: LN_DZ(HNO_ACT_SILU); break;
            default: LN_DZ(HNO_ACT_NONE);
        }
#undef LN_DZ
        HNO_CHECK_LAUNCH();
    }
    const void *d = dz ? (const void *)dz : dy;
    LinArgs a = {};
    a.part = part;
    if (dx) {
        a.A = d; a.lda = N; a.B = w; a.ldb = K; a.y = dx; a.M = M; a.N = K; a.K = N;
        if (int rc = ln_product<T, false, true, HNO_ACT_NONE>(a, s)) return rc;
    }
    a.db_slab = slab; a.db = db; a.db_runs = runs; a.db_n = N; a.db32 = db_dtype == HNO_F32;
    if (dw) {
        a.A = d; a.lda = N; a.B = x; a.ldb = ldx; a.y = dw; a.out32 = sizeof(T) == 2 && dw_dtype == HNO_F32; a.M = N; a.N = K; a.K = M;
        return ln_product<T, true, true, HNO_ACT_NONE>(a, s);
    }
    return db ? ln_bias<T>(a, s) : HNO_OK;
}

extern "C" int hno_linear_bwd(int dtype, const void *dy, const void *z, const void *x, long long ldx, const void *w, void *dx, void *dw, int dw_dtype, void *db,
                              int db_dtype, int M, int N, int K, int act, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = ln_check("hno_linear_bwd", dtype, M, N, K, act)) return rc;
    HNO_REQUIRE(dy && (act == HNO_ACT_NONE || z) && (!dx || w) && (!dw || (x && ldx >= K)) && (dx || dw || db), "hno_linear_bwd: bad argument");
    HNO_REQUIRE(ln_type(dw, dw_dtype, dtype) && ln_type(db, db_dtype, dtype), "hno_linear_bwd: gradients of types %d, %d beside type %d", dw_dtype, db_dtype, dtype);
    const size_t need = hno_linear_workspace_bytes(dtype, M, N, K, act, 1);
    HNO_REQUIRE(workspace && workspace_bytes >= need, "hno_linear_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (dtype == HNO_BF16) return ln_backward<tkh>(dy, z, x, ldx, w, dx, dw, dw_dtype, db, db_dtype, M, N, K, act, (char *)workspace, (hipStream_t)stream);
    return ln_backward<float>(dy, z, x, ldx, w, dx, dw, dw_dtype, db, db_dtype, M, N, K, act, (char *)workspace, (hipStream_t)stream);
}
