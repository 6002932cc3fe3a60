// Softmax attention on (B, T, H, D) tokens, forward and backward (hno_attn_fwd, hno_attn_bwd).
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij) / sum_j exp(s_ij) over the visible keys,  o_i = sum_j p_ij v_j
//   D_i = sum_c do_ic o_ic,  ds_ij = p_ij (do_i . v_j - D_i),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do
//
// Neither p nor ds is written to memory.  The forward pass keeps the running maximum and sum of each row and leaves
// lse_i = log2 sum_j exp(s_ij); the backward kernel recomputes p_ij = 2^(s_ij log2(e) - lse_i).  Some of its workgroups walk the keys for a
// tile of queries (dq), others the queries (of all heads that share the keys) for a tile of keys (dk, dv) -- 7 or 8 products where
// atomic sums would need 5, but every sum has one owner and a fixed order, so results do not change from run to run.
//
// A wave owns 32 rows of its side as the COLUMNS of its products (lane & 31): the softmax statistics are then one value per lane, and the
// registers of a product are the operand of the next (hno_tokens.h).  The other side comes through LDS, row by row as in memory; its
// transposed reads are ds_read_b64_tr_b16.  fp32 tiles lie in LDS as three bf16 ones (hno_tokens.h).
#include "hno_tokens.h"

namespace hno {

struct AttnArgs {
    const void *q, *k, *v, *g, *o, *ores;
    void *out, *outres, *dq, *dk, *dv;
    float *lse, *delta, *part, *part2;
    const unsigned char *mask;
    const int *lens;
    long long qs[3], ks[3], vs[3], ms[4];     // element strides of (batch, token, head); the mask's of (batch, head, query, key)
    int B, Tq, Tk, H, Hk, Dk, Dv, causal, nsplit, tiles, pack, pair, keymask;
    float scale2, scale;                       // scale log2(e), scale
};

constexpr int AT_WAVES = 4, AT_ROWS = 32 * AT_WAVES;
template <typename T> constexpr int at_tile() { return sizeof(T) == 2 ? 64 : 32; }     // rows of the streamed side per step

__device__ __forceinline__ int at_length(const AttnArgs &a, int b) {
    if (!a.lens) return a.Tk;
    const int n = a.lens[b];
    return n < 0 ? 0 : (n > a.Tk ? a.Tk : n);
}
__device__ __forceinline__ float at_other_half(float x) { return __shfl_xor(x, 32); }
__device__ __forceinline__ int at_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }   // result register -> row of the tile

// Where element d (a multiple of 4) of row `row` stands in an LDS tile of DP channels: rows without padding whose 16-byte chunks change places, so
// that 16 consecutive rows read at one chunk (row reads) and 4 consecutive rows read at four neighbouring chunks (transposed reads)
// touch 64 different banks each (measured conflicts: none); with padded rows the transposed reads met 4-way conflicts.
// DP = 96: a row is 3/4 of the banks, rows shift by themselves and the chunks rotate by row / 4; else an exclusive or.
template <int DP>
__device__ __forceinline__ int at_at(int row, int d) {
    const int c = d >> 3;
    int slot;
    if constexpr (DP == 128) slot = c ^ (((row & 3) << 2) | ((row >> 2) & 3));
    else if constexpr (DP == 64) slot = c ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
    else if constexpr (DP == 32) slot = c ^ ((row >> 2) & 3);
    else slot = c + ((row >> 2) & 3) - (c + ((row >> 2) & 3) >= 12 ? 12 : 0);
    return row * DP + slot * 8 + (d & 7);
}
// LDS byte addresses of a lane's fragments in the tile at `base`: r of row lane & 31, channels 16 kk + 8 (lane >> 5) + {0..7}; c of the transposed tile, channel
// 32 dt + (lane & 31), rows 4 (lane >> 5) + {0..3} and 8 rows on.  Other tiles, planes and rows a multiple of 16 away are immediate offsets of the reads, the
// other buffer is a step of all addresses: worked out for each read they were a third of the vector instructions.
template <int DP>
struct AtAddr {
    unsigned r[DP / 16], c[DP / 16];
    __device__ __forceinline__ void init(const tkh *base, int lane) {
        typedef const __attribute__((address_space(3))) tkh *ldsp;
        const unsigned b = (unsigned)(uintptr_t)(ldsp)base;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            r[i] = b + 2 * at_at<DP>(lane & 31, 16 * i + 8 * (lane >> 5));
            c[i] = b + 2 * at_at<DP>(4 * (lane >> 5) + ((lane & 15) >> 2) + 8 * (i & 1), 32 * (i >> 1) + (lane & 16) + 4 * (lane & 3));
        }
    }
    __device__ __forceinline__ void move(int bytes) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) r[i] += bytes, c[i] += bytes;
    }
};
template <typename T, int DP, int PLANE>
__device__ __forceinline__ TkOp<T> at_rows(const AtAddr<DP> &at, int off, int kk) {
    typedef const __attribute__((address_space(3))) tkb8 *lds8;
    TkOp<T> o;
#pragma unroll
    for (int p = 0; p < tk_planes<T>(); ++p) o.p[p].v = *(lds8)(uintptr_t)(at.r[kk] + 2 * (off + p * PLANE));
    return o;
}
template <typename T, int DP, int PLANE>
__device__ __forceinline__ TkOp<T> at_col(const AtAddr<DP> &at, int off, int dt) {
    typedef __attribute__((address_space(3))) tks4 *lds4;
    TkOp<T> o;
#pragma unroll
    for (int p = 0; p < tk_planes<T>(); ++p) {
        const tks4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at.c[2 * dt] + 2 * (off + p * PLANE)));
        const tks4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at.c[2 * dt + 1] + 2 * (off + p * PLANE)));
        o.p[p].v = __builtin_bit_cast(tkb8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return o;
}

// 8 channels of a row (D % 8 == 0, 16-byte aligned: checked by the entry points); channels from D on are zeros
template <typename T>
__device__ __forceinline__ TkFrag<T> at_load8(const T *row, int d, int D) {
    if (d < D) return tk_row(row + d);
    TkFrag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.set(j, 0.f);
    return f;
}

// A workgroup's share of one tile (ROWS rows of a head) of the streamed side on its way to LDS.  Thread t moves the 16-byte (fp32: 32-byte) slots
// t, t + 256, ...  Use: fetch(tile) -> settle(tile) -> barrier -> read it, with the next fetch behind the barrier.
// Rows from `end` on may hold any row of the tensor: their scores are hidden.  Rows whose flag is set in settle() are zeroed: nobody looks at
// them, so they may hold NaN, and 0 x NaN must not reach a sum.
//
// bf16: LDS-DMA (global_load_lds_dwordx4), which needs no registers: with tiles staged through registers dk and dv of 128 channels took 357 of them, and
// spilled when held to two waves per SIMD.  The DMA writes its slots in lane order, so the slot permutation of at_at is applied to the source.
template <typename T, int DP, int ROWS>
struct AtTile;
template <int DP, int ROWS>
struct AtTile<tkh, DP, ROWS> {
    static constexpr int CH = DP / 8, N = ROWS * CH / (64 * AT_WAVES);
    static_assert(ROWS * CH % (64 * AT_WAVES) == 0, "whole slots per thread");
    unsigned off[N];          // byte offset of the slot's source from the tile's first row
    long long st;
    int D;
    __device__ __forceinline__ static int row(int i, int tid) { return (tid + 64 * AT_WAVES * i) / CH; }
    __device__ __forceinline__ static int chunk(int i, int tid) {
        const int s = tid + 64 * AT_WAVES * i, r = s / CH, slot = s - r * CH;
        if constexpr (DP == 128) return slot ^ (((r & 3) << 2) | ((r >> 2) & 3));
        else if constexpr (DP == 64) return slot ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
        else if constexpr (DP == 32) return slot ^ ((r >> 2) & 3);
        else return slot - ((r >> 2) & 3) + (slot < ((r >> 2) & 3) ? 12 : 0);
    }
    __device__ __forceinline__ void init(long long st_, int D_, int tid) {
        st = st_, D = D_;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = chunk(i, tid) * 8;
            off[i] = (unsigned)(row(i, tid) * st + (c < D ? c : 0)) * 2;      // (channels from D on: multiplied by zeros, or never stored)
        }
    }
    __device__ __forceinline__ void fetch(tkh *tile, const tkh *base, int t0, int end, int tid) {
        typedef __attribute__((address_space(3))) tkh *ldsp;
        const tkh *src = base + (long long)t0 * st;
        const unsigned dst = (unsigned)(uintptr_t)(ldsp)tile + (tid >> 6) * 1024;
        if (t0 + ROWS <= end) {
#pragma unroll
            for (int i = 0; i < N; ++i) tk_dma16(src, off[i], dst + i * 4096);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row(i, tid), c = chunk(i, tid) * 8, last = end - 1 - t0;
                tk_dma16(src, (unsigned)((r < last ? r : last) * st + (c < D ? c : 0)) * 2, dst + i * 4096);
            }
        }
    }
    template <typename P>
    __device__ __forceinline__ void settle(tkh *tile, int tid, P dead) const {
        dma_wait<0>();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (dead(i)) *reinterpret_cast<tku4 *>(tile + (tid + 64 * AT_WAVES * i) * 8) = tku4{0, 0, 0, 0};
    }
};
template <int DP, int ROWS>
struct AtTile<float, DP, ROWS> {
    static constexpr int CH = DP / 8, N = (ROWS * CH + 64 * AT_WAVES - 1) / (64 * AT_WAVES);
    TkFrag<float> r[N];
    long long st;
    int D;
    __device__ __forceinline__ static int row(int i, int tid) { return (tid + 64 * AT_WAVES * i) / CH; }
    __device__ __forceinline__ void init(long long st_, int D_, int) { st = st_, D = D_; }
    __device__ __forceinline__ void fetch(tkh *, const float *base, int t0, int end, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = row(i, tid), d = (tid + 64 * AT_WAVES * i - k * CH) * 8, t = t0 + k;
            r[i] = at_load8(base + (long long)(t < end ? t : end - 1) * st, d, D);
        }
    }
    template <typename P>
    __device__ __forceinline__ void settle(tkh *tile, int tid, P dead) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = row(i, tid), d = (tid + 64 * AT_WAVES * i - k * CH) * 8;
            if (dead(i))
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i].set(j, 0.f);
            if (k >= ROWS) continue;
            const TkOp<float> o = tk_op(r[i]);
#pragma unroll
            for (int p = 0; p < 3; ++p) tk_store8(tile + p * ROWS * DP + at_at<DP>(k, d), o.p[p]);
        }
    }
};
// flags of the rows a thread moves, loaded with them
template <typename T, int DP, int ROWS, typename F>
struct AtFlags {
    F f[AtTile<T, DP, ROWS>::N];
    template <typename G>
    __device__ __forceinline__ void load(int t0, int end, int tid, G get) {
#pragma unroll
        for (int i = 0; i < AtTile<T, DP, ROWS>::N; ++i) {
            const int t = t0 + AtTile<T, DP, ROWS>::row(i, tid);
            f[i] = get(t < end ? t : end - 1);
        }
    }
};

// mask bytes of one row for the 4 x 4 keys of a result (j0 = first key of the 32): word u holds keys j0 + 8 u + 4 h + {0..3}.
// The row is read inside [0, Tk) only; keys beyond it are hidden by the row's limit.
struct AtMask { unsigned w[4]; };
__device__ __forceinline__ AtMask at_mask_row(const AttnArgs &a, const unsigned char *row, int j0, int h) {
    AtMask m;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int key = j0 + 8 * u + 4 * h;
        if (a.ms[3] == 1 && key + 3 < a.Tk) {
            __builtin_memcpy(&m.w[u], row + key, 4);
        } else {
            m.w[u] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) m.w[u] |= key + j < a.Tk ? (unsigned)row[(key + j) * a.ms[3]] << (8 * j) : 0u;
        }
    }
    return m;
}
__device__ __forceinline__ bool at_mask_on(const AtMask &m, int e) { return (m.w[e >> 2] >> (8 * (e & 3))) & 0xffu; }

// use(i, load(i)) for i = 0 ... N - 1, the LDS reads DEPTH ahead of the products that take them.  (Left to itself the compiler reads one product ahead, and
// each product waits for most of an LDS access.)  Vector instructions may move across the steps, reads and products may not; with FREE = 4 they may not either.
template <typename T> constexpr int at_ahead() { return sizeof(T) == 2 ? 4 : 2; }
template <int N, int DEPTH, int FREE = 0x406, typename L, typename U>
__device__ __forceinline__ void at_pipe(L load, U use) {
    decltype(load(0)) ring[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH && i < N; ++i) ring[i] = load(i);
    __builtin_amdgcn_sched_barrier(FREE);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        use(i, ring[i % DEPTH]);
        if (i + DEPTH < N) ring[i % DEPTH] = load(i + DEPTH);
        __builtin_amdgcn_sched_barrier(FREE);
    }
}
// acc(32 rows of the tile x 32 own columns) += tile rows . own fragments; `off`: element offset of the tile's first of these rows
template <typename T, int DP, int PLANE>
__device__ __forceinline__ void at_product(tk16 &acc, const AtAddr<DP> &at, int off, const TkOp<T> (&own)[DP / 16]) {
    at_pipe<DP / 16, at_ahead<T>()>([&](int kk) { return at_rows<T, DP, PLANE>(at, off, kk); }, [&](int kk, const TkOp<T> &o) { acc = tk_mma(o, own[kk], acc); });
}
// two independent products, step by step: neither waits for its own last step
template <typename T, int DP, int PLANE>
__device__ __forceinline__ void at_product2(tk16 &x, tk16 &y, const AtAddr<DP> &at, int offx, const TkOp<T> (&ox)[DP / 16], int offy, const TkOp<T> (&oy)[DP / 16]) {
    at_pipe<DP / 8, at_ahead<T>()>([&](int i) { return at_rows<T, DP, PLANE>(at, i & 1 ? offy : offx, i >> 1); },
                                   [&](int i, const TkOp<T> &o) {
                                       if (i & 1) y = tk_mma(o, oy[i >> 1], y);
                                       else x = tk_mma(o, ox[i >> 1], x);
                                   });
}
// acc[dt] += (32 tile rows)^T . w, w being a result over the same rows.  make(e) brings element e of w about: the second half's between the products of the
// first.  bf16: w (a probability or a score gradient) is rounded to the matrix instruction's operand type, the one rounding on the way to the fp32 sum; a
// second bf16 term of it would cost a second product for less than the rounding of the result.
template <typename T, int DP, int PLANE, typename M>
__device__ __forceinline__ void at_accumulate(tk16 (&acc)[DP / 32], const AtAddr<DP> &at, int off, tk16 &w, M make) {
    constexpr int ND = DP / 32;
    const auto pack = [&](int t) {
        TkFrag<T> f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f.set(j, w[8 * t + j]);
        return tk_op(f);
    };
#pragma unroll
    for (int e = 0; e < 8; ++e) make(e);
    TkOp<T> o = pack(0);
    at_pipe<2 * ND, at_ahead<T>(), 4>([&](int i) { return at_col<T, DP, PLANE>(at, off + 16 * (i / ND) * DP, i % ND); },
                                      [&](int i, const TkOp<T> &x) {
                                          const int d = i % ND;
                                          acc[d] = tk_mma(x, o, acc[d]);
                                          if (i < ND) {
#pragma unroll
                                              for (int e = 0; e < 8; ++e)
                                                  if (e >= 8 * d / ND && e < 8 * (d + 1) / ND) make(8 + e);
                                              if (d == ND - 1) o = pack(1);
                                          }
                                      });
}
// LDS buffers of the streamed side: two (one barrier a step), one where two would leave room for a single workgroup per CU
template <typename T, int DP> constexpr int at_buffers() { return sizeof(T) == 4 && DP == 128 ? 1 : 2; }

// store a transposed accumulator (register = channel, lane = row) as row `dst` of a contiguous tensor
template <typename T, int DP, typename F>
__device__ __forceinline__ void at_store(T *dst, const tk16 (&acc)[DP / 32], int D, int h, F value) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = 32 * dt + 8 * u + 4 * h;
            if (d >= D) continue;
            if constexpr (sizeof(T) == 2) {
                tks4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (short)tk_down<T>(value(acc[dt][4 * u + j]));
                *reinterpret_cast<tks4 *>(dst + d) = w;
            } else {
                tkf4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = value(acc[dt][4 * u + j]);
                *reinterpret_cast<tkf4 *>(dst + d) = w;
            }
        }
}

// Workgroup -> work.  The 8 XCDs take workgroups in turn and each has its own L2: every XCD gets one run of the list
// key head x batch x tile x (head of the group, split), so the workgroups that stream the same keys (or queries) share an L2, and an XCD
// meets batch entries of several lengths.  A causal mask makes tiles unequal: those that see most come first, or, where all workgroups are resident at
// once (pair), each takes a long one and its short counterpart one after the other.
struct AtBlock {
    int b, hk, tile, gi, sp;
};
__device__ __forceinline__ AtBlock at_block(const AttnArgs &a, int grp, int id, int n) {
    const int xcd = id & 7, each = n >> 3, more = n & 7;
    int at = xcd * each + min(xcd, more) + (id >> 3);
    AtBlock w;
    w.sp = at % a.nsplit, at /= a.nsplit;
    w.gi = at % grp, at /= grp;
    const int tiles = a.pair ? (a.tiles + 1) >> 1 : a.tiles;
    w.tile = at % tiles, at /= tiles;
    w.b = at % a.B;
    w.hk = at / a.B;
    return w;
}
// the tile of pass `half` (0, 1) of a workgroup; -1: none.  `back`: the last tile is the one that sees most
__device__ __forceinline__ int at_tile_of(const AttnArgs &a, int t, int half, bool back) {
    if (half && (!a.pair || 2 * t == a.tiles - 1)) return -1;
    return (half != 0) != back ? a.tiles - 1 - t : t;
}
// ------------------------------------------------------------------ rows of the query side
// Where few new tokens share a key head (pack), the rows of all its query heads form one list, so
// the keys are read once: row r stands for query r % Tq of head hb + r / Tq.
struct AtRow {
    int head, i, lim;       // query head, query, and the first key that it does not see
    bool valid;
};
__device__ __forceinline__ AtRow at_query_row(const AttnArgs &a, int r, int hb, int nrows, int L) {
    AtRow w;
    w.valid = r < nrows;
    const int rr = w.valid ? r : nrows - 1, gi = rr / a.Tq;
    w.head = hb + gi;
    w.i = rr - gi * a.Tq;
    const int lim = a.causal ? w.i + L - a.Tq + 1 : L;
    w.lim = !w.valid ? 0 : (lim < L ? lim : L);
    return w;
}
// keys [j0, j1) of this workgroup's split: whole tiles, the same number in each split but the last
__device__ __forceinline__ void at_key_range(const AttnArgs &a, int L, int last_row, int nrows, int sp, int tile, int &j0, int &j1) {
    int end = L;
    if (a.causal && nrows <= a.Tq) {          // (a packed list holds the last query of every head)
        const int e = last_row + L - a.Tq + 1;
        end = e < 0 ? 0 : (e < L ? e : L);
    }
    const int nt = (end + tile - 1) / tile, per = (nt + a.nsplit - 1) / a.nsplit;
    j0 = sp * per * tile;
    j1 = j0 + per * tile;
    if (j1 > end) j1 = end;
}

// the smallest limit of the wave's rows: tiles that end before it need no comparison
__device__ __forceinline__ int at_wave_min(int x) {
#pragma unroll
    for (int k = 16; k; k >>= 1) x = min(x, __shfl_xor(x, k));
    return __builtin_amdgcn_readfirstlane(x);
}
// the weights of 8 keys as an operand (bf16: rounded once, as the matrix instruction takes them), and their sum as the product takes them: the weights of a row then
// add up to one whatever they were rounded to.  With the rounding of the result the error is sqrt(2) of a rounding in the mean square (0.0024, 0.0017 for one).
__device__ __forceinline__ void at_weights(TkFrag<tkh> &f, const tk16 &s, int t, float &l) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f.set(j, s[8 * t + j]);
        f.set(j + 1, s[8 * t + j + 1]);
        l = __builtin_amdgcn_fdot2_f32_bf16(b2{f.v[j], f.v[j + 1]}, one, l, false);
    }
}
__device__ __forceinline__ void at_weights(TkFrag<float> &f, const tk16 &s, int t, float &l) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        f.v[j] = s[8 * t + j];
        l += f.v[j];
    }
}

// Per tile of 32 rows x 32 keys: D / 8 matrix instructions (fp32: six times as many) and about 100 vector ones, the exponentials among them at a quarter of the
// rate; both are bounds.  bf16 2x8x8192x64: 258 us = 1065 TFLOP/s (matrix pipes 38 % busy, vector pipes 54 %), causal 2x16x4096x128: 172 us = 800 TFLOP/s
// of what is visible (41 % and 38 %, two waves a SIMD); fp32 4x1960x96: 46 us = 128 TFLOP/s.  New tokens against a long cache: bound by reading it
// (4 sequences of about 6000 keys, 4 key heads of 128 channels: 16 us, and 4 for the join).
template <typename T, int DP, bool MASK>
__global__ __launch_bounds__(64 * AT_WAVES, sizeof(T) == 4 ? (DP <= 96 ? 2 : 1) : (DP <= 64 ? 3 : 2)) void attn_fwd_kernel(AttnArgs a) {
    constexpr int KT = at_tile<T>(), PLANE = KT * DP, NB = at_buffers<T, DP>();
    constexpr int TILE = tk_planes<T>() * PLANE, V = NB * TILE;             // LDS: the buffers of the keys, then those of the values
    __shared__ __attribute__((aligned(16))) tkh smem[2 * NB * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const AtBlock w0 = at_block(a, a.pack ? 1 : a.H / a.Hk, blockIdx.x, gridDim.x);
    const int b = w0.b, sp = w0.sp, grp = a.H / a.Hk, hk = w0.hk, hb = hk * grp + w0.gi, nrows = a.pack ? grp * a.Tq : a.Tq;
    const int L = at_length(a, b);
    for (int half = 0; half < 2; ++half) {
    const int tile = at_tile_of(a, w0.tile, half, a.causal);
    if (tile < 0) break;
    if (half) __syncthreads();
    const int r0 = tile * AT_ROWS, r = r0 + wave * 32 + (lane & 31);
    const AtRow w = at_query_row(a, r, hb, nrows, L);
    int j0, j1;
    at_key_range(a, L, (r0 + AT_ROWS < nrows ? r0 + AT_ROWS : nrows) - 1, nrows, sp, KT, j0, j1);
    const int lim_all = MASK ? 0 : at_wave_min(w.lim), lim_any = -at_wave_min(-w.lim);

    TkOp<T> qf[DP / 16];
    const T *qrow = (const T *)a.q + b * a.qs[0] + (long long)w.i * a.qs[1] + w.head * a.qs[2];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) qf[kk] = tk_op(at_load8(qrow, 16 * kk + 8 * h, a.Dk));
    const T *kb = (const T *)a.k + b * a.ks[0] + hk * a.ks[2], *vb = (const T *)a.v + b * a.vs[0] + hk * a.vs[2];
    const unsigned char *mrow = MASK ? a.mask + b * a.ms[0] + w.head * a.ms[1] + (long long)w.i * a.ms[2] : nullptr;
    // a mask that hides a key from every query of this workgroup takes the value row out too: 0 x NaN would be NaN
    const unsigned char *mkey = MASK && a.keymask ? a.mask + b * a.ms[0] + hb * a.ms[1] : nullptr;
    AtTile<T, DP, KT> ks, vs;
    AtFlags<T, DP, KT, unsigned char> flag;
    ks.init(a.ks[1], a.Dk, tid);
    vs.init(a.vs[1], a.Dv, tid);
    const auto fetch = [&](int to, int j) {
        ks.fetch(smem + to * TILE, kb, j, j1, tid);
        vs.fetch(smem + V + to * TILE, vb, j, j1, tid);
        if (MASK && mkey) flag.load(j, j1, tid, [&](int t) { return mkey[t * a.ms[3]]; });
    };
    const auto settle = [&](int to) {
        ks.settle(smem + to * TILE, tid, [](int) { return false; });
        vs.settle(smem + V + to * TILE, tid, [&](int i) { return MASK && mkey && !flag.f[i]; });
    };

    tk16 acc[DP / 32] = {};
    float m = -INFINITY, l = 0.f, shift = 0.f;
    const float slack = 8.f / a.scale2;           // the maximum is raised, and the sums rescaled, only where weights would exceed 2^8
    AtAddr<DP> at;
    at.init(smem, lane);
    int buf = 0;
    if (j0 < j1) fetch(0, j0);
    for (int j = j0; j < j1; j += KT, buf ^= NB - 1, at.move(NB == 1 ? 0 : (buf ? 2 * TILE : -2 * TILE))) {
        if (NB == 1) __syncthreads();
        settle(buf);
        __syncthreads();
        if (j + KT < j1) fetch(buf ^ (NB - 1), j + KT);
        if (j >= lim_any) continue;             // none of this wave's rows sees the tile
        tk16 s[KT / 32] = {};
        AtMask mk[KT / 32];
        if (MASK)
#pragma unroll
            for (int n = 0; n < KT / 32; ++n) mk[n] = at_mask_row(a, mrow, j + 32 * n, h);
        if constexpr (KT == 64) at_product2<T, DP, PLANE>(s[0], s[1], at, 0, qf, 32 * DP, qf);
        else at_product<T, DP, PLANE>(s[0], at, 0, qf);
        if (j + KT > lim_all) {
            asm volatile("");               // (a branch: the comparisons are not to be made for whole tiles)
#pragma unroll
            for (int n = 0; n < KT / 32; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool on = j + 32 * n + at_row(e, h) < w.lim && (!MASK || at_mask_on(mk[n], e));
                    s[n][e] = on ? s[n][e] : -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < KT / 32; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[n][e]);
        top = fmaxf(top, at_other_half(top));
        if (__any(top > m + slack)) {
            const float up = fmaxf(m, top), old = __builtin_amdgcn_exp2f((m - (up == -INFINITY ? 0.f : up)) * a.scale2);
            m = up;
            shift = up == -INFINITY ? 0.f : up * a.scale2;
            l *= old;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= old;
        }
        // the weights of 8 keys at a time, those of the next 8 between the products of these (2x8x8192x64: 258 us, with all of them in front 273)
        constexpr int ND = DP / 32, G = KT / 16;
        const auto weigh = [&](int g, int e0, int e1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= e0 && e < e1) s[g >> 1][8 * (g & 1) + e] = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + e], a.scale2, -shift));
        };
        const auto pack = [&](int g) {
            TkFrag<T> f;
            at_weights(f, s[g >> 1], g & 1, l);
            return tk_op(f);
        };
        weigh(0, 0, 8);
        TkOp<T> o = pack(0);
        at_pipe<G * ND, at_ahead<T>(), 4>([&](int i) { return at_col<T, DP, PLANE>(at, V + 16 * (i / ND) * DP, i % ND); },
                                          [&](int i, const TkOp<T> &x) {
                                              const int g = i / ND, d = i % ND;
                                              acc[d] = tk_mma(x, o, acc[d]);
                                              if (g + 1 < G) {
                                                  weigh(g + 1, 8 * d / ND, 8 * (d + 1) / ND);
                                                  if (d == ND - 1) o = pack(g + 1);
                                              }
                                          });
    }
    l += at_other_half(l);
    if (!w.valid) continue;
    const long long row = ((long long)b * a.Tq + w.i) * a.H + w.head;
    if (a.nsplit > 1) {
        const long long rows = (long long)a.B * a.Tq * a.H, at = sp * rows + row;
        at_store<float, DP>(a.part + at * a.Dv, acc, a.Dv, h, [](float x) { return x; });
        if (h == 0) {
            a.part2[2 * at] = m == -INFINITY ? m : m * a.scale2;
            a.part2[2 * at + 1] = l;
        }
        continue;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    at_store<T, DP>((T *)a.out + row * a.Dv, acc, a.Dv, h, [&](float x) { return x * inv; });
    if (sizeof(T) == 2 && a.outres)     // what the rounding of o lost: the backward pass needs D_i = do . o to more than 8 bits
        at_store<T, DP>((T *)a.outres + row * a.Dv, acc, a.Dv, h,
                        [&](float x) { const float y = x * inv; return y - tk_up(tk_down<T>(y)); });
    if (a.lse && h == 0) a.lse[row] = m == -INFINITY ? INFINITY : m * a.scale2 + __builtin_amdgcn_logf(l);   // +inf: an empty row
    }
}

// joins the splits of a row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  32 lanes of 4 channels; the 8 groups of lanes share the splits of one
// row (many splits, few rows: 32 splits of 64 rows took 35 us with one wave per row) or take a row each.  Each lane loads its (at most 8)
// splits at once.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const float *__restrict__ part, const float *__restrict__ ml, T *__restrict__ out,
                                                        T *__restrict__ outres, float *__restrict__ lse, long long rows, int Dv, int nsplit) {
    __shared__ tkf4 sum[8][32];
    __shared__ float wsum[8][32], top[8][32];
    const int c = threadIdx.x & 31, y = threadIdx.x >> 5, ys = nsplit > 8 ? 8 : 1, s0 = ys > 1 ? y : 0;
    const long long row = ys > 1 ? blockIdx.x : (long long)blockIdx.x * 8 + y;
    const bool on = row < rows, in = on && 4 * c < Dv;
    float ms[8], ls[8], m = -INFINITY, l = 0.f;
    tkf4 xs[8], x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int s = s0 + k * ys;
        const long long at = s * rows + row;
        ms[k] = on && s < nsplit ? ml[2 * at] : -INFINITY;
        ls[k] = on && s < nsplit ? ml[2 * at + 1] : 0.f;
        xs[k] = in && s < nsplit ? *reinterpret_cast<const tkf4 *>(part + at * Dv + 4 * c) : tkf4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, ms[k]);
    const float shift = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float f = __builtin_amdgcn_exp2f(ms[k] - shift);
        l = fmaf(f, ls[k], l);
        x += f * xs[k];
    }
    if (ys > 1) {
        sum[y][c] = x, wsum[y][c] = l, top[y][c] = m;
        __syncthreads();
        if (y) return;
        float all = m;
        for (int k = 1; k < 8; ++k) all = fmaxf(all, top[k][c]);
        const float base = all == -INFINITY ? 0.f : all;
        x = tkf4{0.f, 0.f, 0.f, 0.f}, l = 0.f;
        for (int k = 0; k < 8; ++k) {
            const float f = __builtin_amdgcn_exp2f(top[k][c] - base);
            l = fmaf(f, wsum[k][c], l);
            x += f * sum[k][c];
        }
        m = all;
    }
    if (!on) return;
    if (lse && c == 0) lse[row] = m == -INFINITY ? INFINITY : m + __builtin_amdgcn_logf(l);
    if (!in) return;
    x *= l == 0.f ? 0.f : 1.f / l;
    if constexpr (sizeof(T) == 2) {
        tks4 t, r;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            t[j] = (short)tk_down<T>(x[j]);
            r[j] = (short)tk_down<T>(x[j] - tk_up((T)t[j]));
        }
        *reinterpret_cast<tks4 *>(out + row * Dv + 4 * c) = t;
        if (outres) *reinterpret_cast<tks4 *>(outres + row * Dv + 4 * c) = r;
    } else {
        *reinterpret_cast<tkf4 *>(out + row * Dv + 4 * c) = x;
    }
}

// D_i = sum_c do_ic o_ic.  16 lanes per row.
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(const T *__restrict__ g, const T *__restrict__ o, const T *__restrict__ ores,
                                                         const float *__restrict__ lse, float *__restrict__ delta, long long rows, int D) {
    const long long row = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int c = threadIdx.x & 15;
    float s = 0.f;
    if (row < rows && lse[row] != INFINITY)
        if (const int d = 8 * c; d < D) {
            const TkFrag<T> x = tk_row(g + row * D + d), y = tk_row(o + row * D + d);
            TkFrag<T> z = y;
            if (ores) z = tk_row(ores + row * D + d);
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf((float)x.v[j], ores ? (float)y.v[j] + (float)z.v[j] : (float)y.v[j], s);
        }
#pragma unroll
    for (int k = 8; k; k >>= 1) s += __shfl_xor(s, k);
    if (row < rows && c == 0) delta[row] = s;
}

// LDS of a backward workgroup: the streamed side's two tensors, then lse and D of their rows
template <typename T, int DP> constexpr int at_half() { return at_buffers<T, DP>() * tk_planes<T>() * at_tile<T>() * DP; }

// dq of a tile of queries
template <typename T, int DP, bool MASK>
__device__ __forceinline__ void at_dq(const AttnArgs &a, const AtBlock &w0, tkh *smem) {
    constexpr int KT = at_tile<T>(), PLANE = KT * DP, NB = at_buffers<T, DP>();
    constexpr int TILE = tk_planes<T>() * PLANE, V = at_half<T, DP>();
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int b = w0.b, sp = w0.sp, grp = a.H / a.Hk, hk = w0.hk, hb = hk * grp + w0.gi, nrows = a.pack ? grp * a.Tq : a.Tq;
    const int L = at_length(a, b);
    for (int half = 0; half < 2; ++half) {
    const int tile = at_tile_of(a, w0.tile, half, a.causal);
    if (tile < 0) break;
    if (half) __syncthreads();
    const int r0 = tile * AT_ROWS, r = r0 + wave * 32 + (lane & 31);
    const AtRow w = at_query_row(a, r, hb, nrows, L);
    int j0, j1;
    at_key_range(a, L, (r0 + AT_ROWS < nrows ? r0 + AT_ROWS : nrows) - 1, nrows, sp, KT, j0, j1);
    const long long row = ((long long)b * a.Tq + w.i) * a.H + w.head;
    TkOp<T> qf[DP / 16], gf[DP / 16];
    const T *qrow = (const T *)a.q + b * a.qs[0] + (long long)w.i * a.qs[1] + w.head * a.qs[2], *grow = (const T *)a.g + row * a.Dv;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        qf[kk] = tk_op(at_load8(qrow, 16 * kk + 8 * h, a.Dk));
        gf[kk] = tk_op(at_load8(grow, 16 * kk + 8 * h, a.Dv));
    }
    const float lse = a.lse[row], delta = a.delta[row];
    const T *kb = (const T *)a.k + b * a.ks[0] + hk * a.ks[2], *vb = (const T *)a.v + b * a.vs[0] + hk * a.vs[2];
    const unsigned char *mrow = MASK ? a.mask + b * a.ms[0] + w.head * a.ms[1] + (long long)w.i * a.ms[2] : nullptr;
    const unsigned char *mkey = MASK && a.keymask ? a.mask + b * a.ms[0] + hb * a.ms[1] : nullptr;
    const int lim_all = MASK ? 0 : at_wave_min(w.lim), lim_any = -at_wave_min(-w.lim);
    AtTile<T, DP, KT> ks, vs;
    AtFlags<T, DP, KT, unsigned char> flag;
    ks.init(a.ks[1], a.Dk, tid);
    vs.init(a.vs[1], a.Dv, tid);
    const auto fetch = [&](int to, int j) {
        ks.fetch(smem + to * TILE, kb, j, j1, tid);
        vs.fetch(smem + V + to * TILE, vb, j, j1, tid);
        if (MASK && mkey) flag.load(j, j1, tid, [&](int t) { return mkey[t * a.ms[3]]; });
    };
    const auto settle = [&](int to) {
        ks.settle(smem + to * TILE, tid, [&](int i) { return MASK && mkey && !flag.f[i]; });
        vs.settle(smem + V + to * TILE, tid, [](int) { return false; });
    };
    tk16 acc[DP / 32] = {};
    AtAddr<DP> at;
    at.init(smem, lane);
    int buf = 0;
    if (j0 < j1) fetch(0, j0);
    for (int j = j0; j < j1; j += KT, buf ^= NB - 1, at.move(NB == 1 ? 0 : (buf ? 2 * TILE : -2 * TILE))) {
        if (NB == 1) __syncthreads();
        settle(buf);
        __syncthreads();
        if (j + KT < j1) fetch(buf ^ (NB - 1), j + KT);
        if (j >= lim_any) continue;             // none of this wave's rows sees the tile
        const bool whole = j + KT <= lim_all;
#pragma unroll
        for (int n = 0; n < KT / 32; ++n) {
            AtMask mk;
            if (MASK) mk = at_mask_row(a, mrow, j + 32 * n, h);
            tk16 s = {}, dp = {};
            at_product2<T, DP, PLANE>(s, dp, at, 32 * n * DP, qf, V + 32 * n * DP, gf);
            if (!whole) {
                asm volatile("");           // (a branch: the comparisons are not to be made for whole tiles)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool on = j + 32 * n + at_row(e, h) < w.lim && (!MASK || at_mask_on(mk, e));
                    s[e] = on ? s[e] : -INFINITY;
                    dp[e] = on ? dp[e] : 0.f;           // (whatever a hidden value holds)
                }
            }
            at_accumulate<T, DP, PLANE>(acc, at, 32 * n * DP, s,
                                        [&](int e) { s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, -lse)) * (dp[e] - delta); });
        }
    }
    if (!w.valid) continue;
    if (a.nsplit > 1) {
        const long long rows = (long long)a.B * a.Tq * a.H;
        at_store<float, DP>(a.part + (sp * rows + row) * a.Dk, acc, a.Dk, h, [&](float x) { return x * a.scale; });
        continue;
    }
    at_store<T, DP>((T *)a.dq + row * a.Dk, acc, a.Dk, h, [&](float x) { return x * a.scale; });
    }
}

// dk (WHAT & 1) and dv (WHAT & 2) of a tile of keys
template <typename T, int DP, bool MASK, int WHAT>
__device__ __forceinline__ void at_dkv(const AttnArgs &a, const AtBlock &w0, tkh *smem) {
    constexpr int QT = at_tile<T>(), PLANE = QT * DP, NB = at_buffers<T, DP>();
    constexpr int TILE = tk_planes<T>() * PLANE, G = at_half<T, DP>();
    typedef float Rows[NB][QT];
    Rows &lses = *reinterpret_cast<Rows *>(smem + 2 * at_half<T, DP>()), &deltas = *reinterpret_cast<Rows *>(smem + 2 * at_half<T, DP>() + 2 * NB * QT);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int b = w0.b, sp = w0.sp, grp = a.H / a.Hk, hk = w0.hk;
    const int L = at_length(a, b), off = L - a.Tq;
    for (int half = 0; half < 2; ++half) {
    const int ktile = at_tile_of(a, w0.tile, half, false);
    if (ktile < 0) break;
    if (half) __syncthreads();
    const int key0 = ktile * AT_ROWS, key = key0 + wave * 32 + (lane & 31);
    const bool valid = key < a.Tk;
    const int kc = valid ? key : a.Tk - 1;
    // queries that see this key: [first, Tq)
    const int first = key >= L ? 0x7fffffff : (a.causal ? key - off : 0);
    constexpr bool DK = WHAT & 1, DV = WHAT & 2;
    TkOp<T> kf[DP / 16], vf[DP / 16];
    const T *krow = (const T *)a.k + b * a.ks[0] + (long long)kc * a.ks[1] + hk * a.ks[2];
    const T *vrow = (const T *)a.v + b * a.vs[0] + (long long)kc * a.vs[1] + hk * a.vs[2];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        kf[kk] = tk_op(at_load8(krow, 16 * kk + 8 * h, a.Dk));
        if (DK) vf[kk] = tk_op(at_load8(vrow, 16 * kk + 8 * h, a.Dv));
    }
    tk16 acck[DK ? DP / 32 : 1] = {}, accv[DV ? DP / 32 : 1] = {};
    // the list of (head of the group, query tile) that sees any key of this tile, cut into nsplit runs
    int qt0 = a.causal && key0 - off > 0 ? (key0 - off) / QT : 0;
    const int nqt = (a.Tq + QT - 1) / QT;
    if (key0 >= L || qt0 > nqt) qt0 = nqt;
    const int each = nqt - qt0, total = each * grp, per = (total + a.nsplit - 1) / a.nsplit;
    const int it1 = (sp + 1) * per < total ? (sp + 1) * per : total;
    // queries from here on are seen by every key of the wave
    const int first_all = MASK || key0 + wave * 32 + 32 > L ? 0x7fffffff : (a.causal ? key0 + wave * 32 + 31 - off : 0);
    AtTile<T, DP, QT> qs, gs;
    AtFlags<T, DP, QT, float> flag;
    qs.init(a.qs[1], a.Dk, tid);
    gs.init((long long)a.H * a.Dv, a.Dv, tid);
    float nlse = 0.f, ndelta = 0.f;               // row tid of the tile
    const float unscale = -1.f / a.scale2;
    const int empty = a.causal ? -off : 0;        // queries before it see nothing
    int i_next = 0;
    const auto fetch = [&](int to, int gi, int qt) {
        const int i0 = qt * QT, head = hk * grp + gi;
        const long long row0 = ((long long)b * a.Tq) * a.H + head;
        i_next = i0;
        qs.fetch(smem + to * TILE, (const T *)a.q + b * a.qs[0] + head * a.qs[2], i0, a.Tq, tid);
        gs.fetch(smem + G + to * TILE, (const T *)a.g + row0 * a.Dv, i0, a.Tq, tid);
        if (MASK) flag.load(i0, a.Tq, tid, [&](int t) { return a.lse[row0 + (long long)t * a.H]; });
        if (tid < QT) {
            const int i = i0 + tid < a.Tq ? i0 + tid : a.Tq - 1;
            nlse = a.lse[row0 + (long long)i * a.H];
            ndelta = a.delta[row0 + (long long)i * a.H];
        }
    };
    const auto settle = [&](int to) {
        // queries that see nothing, by their position or by the mask
        const auto dead = [&](int i) { return i_next + AtTile<T, DP, QT>::row(i, tid) < empty || (MASK && flag.f[i] == INFINITY); };
        qs.settle(smem + to * TILE, tid, dead);
        gs.settle(smem + G + to * TILE, tid, dead);
        if (tid < QT) lses[to][tid] = sizeof(T) == 2 ? nlse * unscale : -nlse, deltas[to][tid] = -ndelta;
    };
    AtAddr<DP> at;
    at.init(smem, lane);
    int buf = 0;
    int gi = each > 0 ? sp * per / each : 0, qt = qt0 + sp * per - gi * each;
    if (sp * per < it1) fetch(0, gi, qt);
    for (int it = sp * per; it < it1; ++it, buf ^= NB - 1, at.move(NB == 1 ? 0 : (buf ? 2 * TILE : -2 * TILE))) {
        if (NB == 1) __syncthreads();
        settle(buf);
        __syncthreads();
        const int i0 = qt * QT, head = hk * grp + gi;
        if (++qt == nqt) qt = qt0, ++gi;
        if (it + 1 < it1) fetch(buf ^ (NB - 1), gi, qt);
        const bool whole = i0 >= first_all && i0 + QT <= a.Tq;
        const unsigned char *mcol = MASK ? a.mask + b * a.ms[0] + head * a.ms[1] + kc * a.ms[3] : nullptr;
#pragma unroll
        for (int n = 0; n < QT / 32; ++n) {
            unsigned char mk[16];
            if (MASK)
#pragma unroll
                for (int e = 0; e < 16; ++e) mk[e] = mcol[min(i0 + 32 * n + at_row(e, h), a.Tq - 1) * a.ms[2]];
            // bf16: the products start at -lse / (scale log2 e) and -D (fp32 would lose bits of s to them)
            constexpr bool START = sizeof(T) == 2;
            tk16 s = {}, dp = {};
            const auto rows4 = [&](const float *x, int e) { return *reinterpret_cast<const tkf4 *>(x + 32 * n + 2 * e + 4 * h); };       // e: a multiple of 4
            if constexpr (START)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const tkf4 le = rows4(lses[buf], e), de = DK ? rows4(deltas[buf], e) : tkf4{};
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[e + j] = le[j], dp[e + j] = de[j];
                }
            if constexpr (DK) at_product2<T, DP, PLANE>(s, dp, at, 32 * n * DP, kf, G + 32 * n * DP, vf);
            else at_product<T, DP, PLANE>(s, at, 32 * n * DP, kf);
            if constexpr (!START)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const tkf4 le = rows4(lses[buf], e), de = rows4(deltas[buf], e);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[e + j] = fmaf(s[e + j], a.scale2, le[j]), dp[e + j] += de[j];
                }
            if (!whole) {
                asm volatile("");           // (a branch: the comparisons are not to be made for whole tiles)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int i = i0 + 32 * n + at_row(e, h);
                    const bool on = i >= first && i < a.Tq && (!MASK || mk[e]);
                    s[e] = on ? s[e] : -INFINITY;
                    if (DK) dp[e] = on ? dp[e] : 0.f;
                }
            }
            const auto make = [&](int e) {
                s[e] = __builtin_amdgcn_exp2f(START ? s[e] * a.scale2 : s[e]);
                if (DK) dp[e] *= s[e];
            };
            if constexpr (DV) at_accumulate<T, DP, PLANE>(accv, at, G + 32 * n * DP, s, make);
            if constexpr (DK) at_accumulate<T, DP, PLANE>(acck, at, 32 * n * DP, dp, [&](int e) { if (!DV) make(e); });
        }
    }
    if (!valid) continue;
    const long long row = ((long long)b * a.Tk + key) * a.Hk + hk;
    if (a.nsplit > 1) {
        const long long at = sp * ((long long)a.B * a.Tk * a.Hk) + row;
        if constexpr (DK) at_store<float, DP>(a.part + at * a.Dk, acck, a.Dk, h, [&](float x) { return x * a.scale; });
        if constexpr (DV) at_store<float, DP>(a.part2 + at * a.Dv, accv, a.Dv, h, [](float x) { return x; });
        continue;
    }
    if constexpr (DK) at_store<T, DP>((T *)a.dk + row * a.Dk, acck, a.Dk, h, [&](float x) { return x * a.scale; });
    if constexpr (DV) at_store<T, DP>((T *)a.dv + row * a.Dv, accv, a.Dv, h, [](float x) { return x; });
    }
}

// The three gradients in one launch: the runs of workgroups stand one behind the other in the grid, each padded to whole rounds of the XCDs, dk and dq
// (three products) before dv (two).  dk and dv are one workgroup's work where the registers of both leave two waves per SIMD (bf16 up to 64 channels) or one wave
// is all there is anyway (fp32), else two's.  Two waves with a few spilled registers are better than one with none: masked, 128 channels, 320 us against 379.
// bf16 causal 2x16x4096x128 (4 key heads): 653 us, 840 TFLOP/s of the 8 products it forms, 525 of the 5 that the gradients need; matrix pipes 47 % busy, vector
// pipes 34 %.  fp32 4x1960x96: 145 us.
template <typename T, int DP> constexpr bool at_joint() { return sizeof(T) == 4 || DP <= 64; }
template <typename T, int DP, bool MASK>
__global__ __launch_bounds__(64 * AT_WAVES, sizeof(T) == 2 ? 2 : 1) void attn_bwd_kernel(AttnArgs aq, AttnArgs ak, int nq, int nk) {
    __shared__ __attribute__((aligned(16))) tkh smem[2 * at_half<T, DP>() + 4 * at_buffers<T, DP>() * at_tile<T>()];
    const int nq8 = (nq + 7) & ~7, nk8 = (nk + 7) & ~7;
    int id = blockIdx.x;
    if (id < nk8) {
        if (id < nk) at_dkv<T, DP, MASK, at_joint<T, DP>() ? 3 : 1>(ak, at_block(ak, 1, id, nk), smem);
        return;
    }
    id -= nk8;
    if (id < nq8) {
        if (id < nq) at_dq<T, DP, MASK>(aq, at_block(aq, aq.pack ? 1 : aq.H / aq.Hk, id, nq), smem);
        return;
    }
    id -= nq8;
    if constexpr (!at_joint<T, DP>())
        if (id < nk) at_dkv<T, DP, MASK, 2>(ak, at_block(ak, 1, id, nk), smem);
}

// out = sum over splits, in split order, of up to three tensors (4 elements a thread; n is a multiple of 8)
struct AtSum {
    const float *part[3];
    void *out[3];
    long long n[3];
    int nsplit[3];
};
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(AtSum a) {
    long long i = 4 * ((long long)blockIdx.x * 256 + threadIdx.x);
    int k = 0;
    while (k < 2 && i >= a.n[k]) i -= a.n[k++];
    const long long n = a.n[k];
    if (i >= n) return;
    const float *p = a.part[k] + i;
    tkf4 x = *reinterpret_cast<const tkf4 *>(p);
#pragma unroll 4
    for (int s = 1; s < a.nsplit[k]; ++s) x += *reinterpret_cast<const tkf4 *>(p + s * n);
    if constexpr (sizeof(T) == 2) {
        tks4 t;
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = (short)tk_down<T>(x[j]);
        *reinterpret_cast<tks4 *>((T *)a.out[k] + i) = t;
    } else {
        *reinterpret_cast<tkf4 *>((T *)a.out[k] + i) = x;
    }
}

}  // namespace hno

using namespace hno;

// how many runs the streamed side is cut into: two workgroups per CU, no run shorter than `least` tiles; where that is not to be had, one per CU and runs of
// two tiles.  The backward kernel holds three gradients' workgroups: causal 2x16x4096x128 takes 12 % longer in runs of two than in the four that this rule gives,
// while 3x6x777x1033x80 takes 69 us with one workgroup per CU and gradient (135 with two, in launches of their own).
static int at_splits(long long groups, long long steps, int least) {
    if (groups < 1) return 1;                                  // no keys at all
    long long n = groups >= 512 ? 1 : (512 + groups - 1) / groups;
    if (least > 2 && steps < least * n) n = groups >= 256 ? 1 : (256 + groups - 1) / groups;
    if (n > steps / 2) n = steps / 2;
    if (n > 64) n = 64;
    return n < 1 ? 1 : (int)n;
}
struct AtPlan {
    int pack, q_tiles, q_heads, q_split, q_pair, k_tiles, k_split, k_pair;
    long long q_blocks, k_blocks;
};
static AtPlan at_plan(const hno_attn_t *p, bool backward) {
    AtPlan n;
    const int grp = p->H / p->Hk, KT = p->dtype == HNO_BF16 ? 64 : 32;
    n.pack = grp > 1 && p->Tq < AT_ROWS;
    n.q_tiles = ceil_div(n.pack ? grp * p->Tq : p->Tq, AT_ROWS);
    n.q_heads = n.pack ? p->Hk : p->H;
    n.k_tiles = ceil_div(p->Tk, AT_ROWS);
    long long q = (long long)n.q_heads * p->B, k = (long long)p->Hk * p->B;
    n.q_pair = p->causal && q * n.q_tiles <= 1024;
    n.k_pair = p->causal && k * n.k_tiles <= 1024;
    q *= n.q_pair ? (n.q_tiles + 1) / 2 : n.q_tiles;
    k *= n.k_pair ? (n.k_tiles + 1) / 2 : n.k_tiles;
    // Forward: a few new tokens want all the chip's loads at once (4x1x16x128 against 6000 keys 16 us in 32 runs, a sixth more in 16); a tile of fp32 is so much work
    // that a second workgroup per CU is worth more slabs (4x1960x96: 8 runs 46 + 5.6 us with the join, 4 runs 54 + 4.4), one of bf16 is not
    // (causal 4x4096x128, 1 key head: 8 runs 38.5 + 12.8, 4 runs 43 + 7.8)
    const int q_least = backward ? 16 : (n.q_tiles == 1 ? 2 : (p->dtype == HNO_F32 ? 6 : 16));
    n.q_split = at_splits(q, ceil_div(p->Tk, KT), q_least);
    n.k_split = at_splits(k, (long long)ceil_div(p->Tq, KT) * grp, 16);
    n.q_blocks = q * n.q_split;
    n.k_blocks = k * n.k_split;
    return n;
}
static size_t at_pad(size_t bytes) { return (bytes + 255) / 256 * 256; }

static bool at_aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int at_check(const hno_attn_t *p, const char *what) {
    HNO_REQUIRE(p, "%s: null argument", what);
    HNO_REQUIRE(p->dtype == HNO_F32 || p->dtype == HNO_BF16, "%s: dtype %d is neither HNO_F32 nor HNO_BF16", what, p->dtype);
    HNO_REQUIRE(p->B > 0 && p->Tq > 0 && p->Tk >= 0 && p->H > 0 && p->Hk > 0 && p->Dk > 0 && p->Dv > 0, "%s: bad size", what);
    HNO_REQUIRE(p->H % p->Hk == 0, "%s: %d query heads do not share %d key heads evenly", what, p->H, p->Hk);
    HNO_REQUIRE(p->scale >= 1e-30f && p->scale <= 1e30f, "%s: scale must be positive, from 1e-30 to 1e30", what);
    if (p->Dk > 128 || p->Dv > 128) return fail(HNO_ELIMIT, "%s: head sizes %d, %d exceed 128", what, p->Dk, p->Dv);
    if (p->Tq > (1 << 28) || p->Tk > (1 << 28) || (long long)(p->H / p->Hk) * p->Tq > (1ll << 30)) return fail(HNO_ELIMIT, "%s: too many tokens", what);
    // a grid holds fewer than 2^32 threads: tiles of 128 rows (dk and dv apart) of 256 threads, and 16 threads a row
    if ((double)p->B * p->H * ((double)ceil_div(p->Tq, AT_ROWS) + 2.0 * ceil_div(p->Tk, AT_ROWS)) > 1.6e7 || (double)p->B * p->H * p->Tq > 2.6e8)
        return fail(HNO_ELIMIT, "%s: the grid is too large", what);
    HNO_REQUIRE(p->q && (p->Tk == 0 || (p->k && p->v)), "%s: null pointer", what);
    const int esz = p->dtype == HNO_BF16 ? 2 : 4;
    bool ok = p->Dk % 8 == 0 && p->Dv % 8 == 0 && at_aligned(p->q) && at_aligned(p->k) && at_aligned(p->v);
    for (int i = 0; i < 3; ++i) ok = ok && p->q_stride[i] * esz % 16 == 0 && p->k_stride[i] * esz % 16 == 0 && p->v_stride[i] * esz % 16 == 0;
    HNO_REQUIRE(ok, "%s: head sizes must be multiples of 8 and rows 16-byte aligned", what);
    for (const long long st : {p->q_stride[1], p->k_stride[1], p->v_stride[1], (long long)p->H * p->Dv})     // offsets inside a tile take 32 bits
        HNO_REQUIRE(st >= 0 && st < (1 << 24), "%s: a token stride of %lld elements", what, st);
    return HNO_OK;
}
static AttnArgs at_args(const hno_attn_t *p) {
    AttnArgs a = {};
    a.q = p->q; a.k = p->k; a.v = p->v; a.mask = p->mask; a.lens = p->kv_lens;
    for (int i = 0; i < 3; ++i) a.qs[i] = p->q_stride[i], a.ks[i] = p->k_stride[i], a.vs[i] = p->v_stride[i];
    for (int i = 0; i < 4; ++i) a.ms[i] = p->mask_stride[i];
    a.B = p->B; a.Tq = p->Tq; a.Tk = p->Tk; a.H = p->H; a.Hk = p->Hk; a.Dk = p->Dk; a.Dv = p->Dv; a.causal = p->causal != 0;
    a.keymask = p->mask && p->mask_stride[2] == 0 && p->mask_stride[1] == 0;
    a.scale = p->scale;
    a.scale2 = p->scale * 1.4426950408889634f;
    return a;
}
static double at_bytes(const hno_attn_t *p, int q_tensors, int k_tensors) {
    return (p->dtype == HNO_BF16 ? 2.0 : 4.0) * ((double)p->B * p->Tq * p->H * p->Dk * q_tensors + (double)p->B * p->Tk * p->Hk * p->Dk * k_tensors);
}

// the kernel of one type for the padded head size, with or without a mask
#define AT_LAUNCH(KERNEL, DP, ...)                                                                                 \
    do {                                                                                                           \
        if (p->mask) hipLaunchKernelGGL((KERNEL<T, DP, true>), dim3(n_), dim3(64 * AT_WAVES), 0, s, __VA_ARGS__);  \
        else hipLaunchKernelGGL((KERNEL<T, DP, false>), dim3(n_), dim3(64 * AT_WAVES), 0, s, __VA_ARGS__);         \
    } while (0)
#define AT_DISPATCH(KERNEL, blocks, ...)                                                                           \
    do {                                                                                                           \
        const int dp_ = round_up(p->Dk > p->Dv ? p->Dk : p->Dv, 32);                                               \
        const unsigned n_ = (unsigned)(blocks);                                                                    \
        if (dp_ == 32) AT_LAUNCH(KERNEL, 32, __VA_ARGS__);                                                         \
        else if (dp_ == 64) AT_LAUNCH(KERNEL, 64, __VA_ARGS__);                                                    \
        else if (dp_ == 96) AT_LAUNCH(KERNEL, 96, __VA_ARGS__);                                                    \
        else AT_LAUNCH(KERNEL, 128, __VA_ARGS__);                                                                  \
    } while (0)

template <typename T>
static int at_forward(const hno_attn_t *p, void *out, void *out_res, float *lse, void *workspace, hipStream_t s) {
    const AtPlan n = at_plan(p, false);
    AttnArgs a = at_args(p);
    const long long rows = (long long)p->B * p->Tq * p->H;
    a.out = out; a.outres = out_res; a.lse = lse; a.pack = n.pack; a.nsplit = n.q_split; a.tiles = n.q_tiles, a.pair = n.q_pair;
    a.part = (float *)workspace;
    a.part2 = (float *)((char *)workspace + at_pad((size_t)n.q_split * rows * p->Dv * sizeof(float)));
    ProfScope _ps(KID_ATTN, s, at_bytes(p, 2, 2));
    AT_DISPATCH(attn_fwd_kernel, n.q_blocks, a);
    HNO_CHECK_LAUNCH();
    if (n.q_split > 1) {
        hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)(n.q_split > 8 ? rows : (rows + 7) / 8)), dim3(256), 0, s, (const float *)a.part, (const float *)a.part2,
                           (T *)out, (T *)out_res, lse, rows, p->Dv, n.q_split);
        HNO_CHECK_LAUNCH();
    }
    return HNO_OK;
}

// floats of the backward pass's slabs: dq, dk, dv
struct AtSlabs {
    size_t q, k, v;
};
static AtSlabs at_slabs(const hno_attn_t *p, const AtPlan &n) {
    const size_t rows = (size_t)p->B * p->Tq * p->H, krows = (size_t)p->B * p->Tk * p->Hk, f = sizeof(float);
    return {n.q_split > 1 ? at_pad(n.q_split * rows * p->Dk * f) : 0, n.k_split > 1 ? at_pad(n.k_split * krows * p->Dk * f) : 0,
            n.k_split > 1 ? at_pad(n.k_split * krows * p->Dv * f) : 0};
}

template <typename T>
static int at_backward(const hno_attn_t *p, const void *out, const void *out_res, const float *lse, const void *dout, void *dq, void *dk, void *dv,
                       void *workspace, hipStream_t s) {
    const AtPlan n = at_plan(p, true);
    const AtSlabs slabs = at_slabs(p, n);
    const long long rows = (long long)p->B * p->Tq * p->H, krows = (long long)p->B * p->Tk * p->Hk;
    char *ws = (char *)workspace + at_pad(rows * sizeof(float));
    AttnArgs aq = at_args(p);
    aq.g = dout; aq.lse = const_cast<float *>(lse); aq.delta = (float *)workspace;
    aq.dq = dq; aq.dk = dk; aq.dv = dv;
    AttnArgs ak = aq;
    aq.pack = n.pack; aq.nsplit = n.q_split; aq.tiles = n.q_tiles; aq.pair = n.q_pair;
    aq.part = (float *)ws;
    ak.nsplit = n.k_split; ak.tiles = n.k_tiles; ak.pair = n.k_pair;
    ak.part = (float *)(ws + slabs.q);
    ak.part2 = (float *)(ws + slabs.q + slabs.k);
    ProfScope _ps(KID_ATTN_BWD, s, at_bytes(p, 4, 4));
    hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, s, (const T *)dout, (const T *)out, (const T *)out_res, lse,
                       aq.delta, rows, p->Dv);
    HNO_CHECK_LAUNCH();
    const int nq = dq ? (int)n.q_blocks : 0, nk = dk && p->Tk > 0 ? (int)n.k_blocks : 0, nv = sizeof(T) == 4 || (p->Dk <= 64 && p->Dv <= 64) ? 0 : nk;
    if (nq + nk == 0) return HNO_OK;
    AT_DISPATCH(attn_bwd_kernel, round_up(nk, 8) + round_up(nq, 8) + nv, aq, ak, nq, nk);
    HNO_CHECK_LAUNCH();
    AtSum sum = {};
    if (nq && n.q_split > 1) sum.part[0] = aq.part, sum.out[0] = dq, sum.n[0] = rows * p->Dk, sum.nsplit[0] = n.q_split;
    if (nk && n.k_split > 1) {
        sum.part[1] = ak.part, sum.out[1] = dk, sum.n[1] = krows * p->Dk, sum.nsplit[1] = n.k_split;
        sum.part[2] = ak.part2, sum.out[2] = dv, sum.n[2] = krows * p->Dv, sum.nsplit[2] = n.k_split;
    }
    if (const long long total = sum.n[0] + sum.n[1] + sum.n[2]) {
        hipLaunchKernelGGL((attn_sum_kernel<T>), dim3((unsigned)((total + 1023) / 1024)), dim3(256), 0, s, sum);
        HNO_CHECK_LAUNCH();
    }
    return HNO_OK;
}

extern "C" size_t hno_attn_workspace_bytes(const hno_attn_t *p, int backward) {
    if (at_check(p, "hno_attn_workspace_bytes") != HNO_OK) return 0;
    const AtPlan n = at_plan(p, backward != 0);
    const size_t rows = (size_t)p->B * p->Tq * p->H, f = sizeof(float);
    if (!backward) return n.q_split > 1 ? at_pad(n.q_split * rows * p->Dv * f) + n.q_split * rows * 2 * f : 0;
    const AtSlabs slabs = at_slabs(p, n);
    return at_pad(rows * f) + slabs.q + slabs.k + slabs.v;
}

extern "C" int hno_attn_fwd(const hno_attn_t *p, void *out, void *out_res, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = at_check(p, "hno_attn_fwd")) return rc;
    HNO_REQUIRE(out && at_aligned(out) && at_aligned(out_res), "hno_attn_fwd: out must be a 16-byte aligned tensor");
    const size_t need = hno_attn_workspace_bytes(p, 0);
    HNO_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && at_aligned(workspace))), "hno_attn_fwd: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
    if (p->dtype == HNO_BF16) return at_forward<tkh>(p, out, out_res, lse, workspace, (hipStream_t)stream);
    return at_forward<float>(p, out, nullptr, lse, workspace, (hipStream_t)stream);
}

extern "C" int hno_attn_bwd(const hno_attn_t *p, const void *out, const void *out_res, const float *lse, const void *dout, void *dq, void *dk, void *dv,
                            void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = at_check(p, "hno_attn_bwd")) return rc;
    HNO_REQUIRE(out && lse && dout && (dq || dk) && !dk == !dv, "hno_attn_bwd: null pointer");
    HNO_REQUIRE(at_aligned(out) && at_aligned(out_res) && at_aligned(dout) && at_aligned(dq) && at_aligned(dk) && at_aligned(dv),
                "hno_attn_bwd: tensors must be 16-byte aligned");
    const size_t need = hno_attn_workspace_bytes(p, 1);
    HNO_REQUIRE(workspace_bytes >= need && workspace && at_aligned(workspace), "hno_attn_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (p->dtype == HNO_BF16) return at_backward<tkh>(p, out, out_res, lse, dout, dq, dk, dv, workspace, (hipStream_t)stream);
    return at_backward<float>(p, out, nullptr, lse, dout, dq, dk, dv, workspace, (hipStream_t)stream);
}
