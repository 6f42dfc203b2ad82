// attention.hip — attention over padded sets of RoIs or map cells, forward and backward, on the matrix cores.
//
//   s_ij = scale * q_i . k_j over the keys j that row i may see,  l_i = log sum_j exp s_ij,  p_ij = exp(s_ij - l_i)
//   o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i,  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij do_i,  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// The backward pass recomputes p from q, k and l; nothing of size rows x keys is ever stored.  dq and (dk, dv) come from two
// kernels, each of which owns its outputs: two products of seven are computed twice, but there are no atomics and the result
// has the same bits in every run.  Query heads that share a key head are laid out as one list of rows (row r = head r / n of
// the group, query r % n), so a key tile is read once for all of them and their gradients add up in registers.
//
// Layout of the 32x32 matrix instruction's result: lane l holds column l & 31 and rows 8 (r / 4) + 4 (l / 32) + r % 4.  The
// products are arranged so that the column is what the statistics belong to (S^T = K Q^T in the forward and dq kernels: one
// query per lane) and so that a result feeds the next product as its second operand without moving between lanes: the
// contraction index may be permuted as long as the first operand, read transposed from LDS, is permuted the same way.
#include "common.hpp"
#include <math.h>
#include <type_traits>

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));

#define AT_THREADS 256
#define AT_WAVES 4
#define AT_LOG2E 1.4426950408889634f
#define AT_LN2 0.6931471805599453f

template <typename T> struct at_vec;
template <> struct at_vec<__bf16> { typedef bf16x8 frag; typedef bf16x4 quad; };
template <> struct at_vec<float> { typedef f32x4 frag; typedef f32x4 quad; };

// Operands of the matrix cores: eight contraction values of a lane, lanes 0..31 the first eight of a block of sixteen, lanes
// 32..63 the second.  A value of 32 bits goes in as three of 16: x = h + m + l, each the rounding of what the ones before left, which is
// exact but for numbers that end below 2^-126.  Of the nine products the six from 2^-16 up are formed; what is left out is less than 2^-25 of
// |x y|, half a rounding in 32 bits.  Six instructions of 32 cycles for sixteen contraction values; the 32-bit matrix instruction
// would take 512 cycles for them.
template <typename T> struct at_parts { static constexpr int N = sizeof(T) == 4 ? 3 : 1; };
template <typename T> struct at_op { bf16x8 p[at_parts<T>::N]; };
__device__ __forceinline__ f32x16 at_mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 at_mma(const at_op<__bf16> &a, const at_op<__bf16> &b, f32x16 c) { return at_mfma(a.p[0], b.p[0], c); }
__device__ __forceinline__ f32x16 at_mma(const at_op<float> &a, const at_op<float> &b, f32x16 c)
{
    c = at_mfma(a.p[2], b.p[0], c);
    c = at_mfma(a.p[0], b.p[2], c);
    c = at_mfma(a.p[1], b.p[1], c);
    c = at_mfma(a.p[1], b.p[0], c);
    c = at_mfma(a.p[0], b.p[1], c);
    return at_mfma(a.p[0], b.p[0], c);
}
__device__ __forceinline__ void at_cut(f32x8 x, at_op<__bf16> &o) { o.p[0] = __builtin_convertvector(x, bf16x8); }
// x - h for the two values of a pair: a dot product of two terms with (-1, 0) or (0, -1), exact (as is the difference of the two numbers),
// one instruction where a conversion back and a difference are two.  (-1, 0) comes from a register: as a constant of the
// instruction, which is of 32 bits, -1 would stand in the other half.
__device__ __forceinline__ void at_less(bf16x2 h, float &x, float &y)
{
    u32 c;
    asm("s_mov_b32 %0, 0xbf80" : "=s"(c));
    x = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, c), x, false);
    y = __builtin_amdgcn_fdot2_f32_bf16(h, (bf16x2){(__bf16)0.f, (__bf16)-1.f}, y, false);
}
// the next part of x, which is left with the rest
__device__ __forceinline__ bf16x8 at_next(f32x8 &x)
{
    const bf16x8 h = __builtin_convertvector(x, bf16x8);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float a = x[e], b = x[e + 1];
        at_less((bf16x2){h[e], h[e + 1]}, a, b);
        x[e] = a;
        x[e + 1] = b;
    }
    return h;
}
__device__ __forceinline__ void at_cut(f32x8 x, at_op<float> &o)
{
    o.p[0] = at_next(x);
    o.p[1] = at_next(x);
    o.p[2] = __builtin_convertvector(x, bf16x8);
}
// eight values of a row in memory
__device__ __forceinline__ void at_read(const __bf16 *p, bool in, at_op<__bf16> &o) { o.p[0] = in ? *(const bf16x8 *)p : (bf16x8)(0.f); }
__device__ __forceinline__ void at_read(const float *p, bool in, at_op<float> &o)
{
    const f32x4 a = in ? *(const f32x4 *)p : (f32x4)(0.f), b = in ? *(const f32x4 *)(p + 4) : (f32x4)(0.f);
    at_cut(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), o);
}
// the value of this lane and of the one 32 away, in either order
__device__ __forceinline__ void at_both(float v, float &x, float &y)
{
    typedef u32 u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    x = __uint_as_float(r[0]);
    y = __uint_as_float(r[1]);
}

// A tile of ROWS rows in LDS, DP values wide, a plane of bf16 for each part, in 16-byte chunks whose place inside the row is
// swizzled by the row.  LDS gives 256 bytes a clock to reads; sixteen lanes that read the same chunk of sixteen successive rows, and
// thirty-two that read four chunks of four successive rows (the transposing read), both cover all 256 bytes modulo 256.  Measured on
// 16001 rows x 128: a swizzle for 128 bytes a clock spent 40% of the LDS's active cycles on conflicts.
template <typename T, int DP, int ROWS> struct at_tile {
    static constexpr int RB = DP * 2, CPR = RB / 16, N = at_parts<T>::N, PLANE = ROWS * RB, BYTES = N * PLANE;
    static __device__ __forceinline__ int swz(int row)
    {
        return CPR >= 16 ? ((row & 3) << 2) | ((row >> 2) & 3) : CPR == 8 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }
    // rows of the tile as an operand: row l & 31, chunk 2 g + l / 32
    static __device__ __forceinline__ at_op<T> row(const char *t, int row, int chunk)
    {
        at_op<T> o;
#pragma unroll
        for (int i = 0; i < N; ++i) o.p[i] = *(const bf16x8 *)(t + i * PLANE + at(row, chunk));
        return o;
    }
    // 16 bytes of a row in memory
    static __device__ __forceinline__ void put(char *t, int row, int c16, u32x4 x)
    {
        if (N == 1) { *(u32x4 *)(t + at(row, c16)) = x; return; }
        f32x4 v = __builtin_bit_cast(f32x4, x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bf16x4 h = __builtin_convertvector(v, bf16x4);
            *(bf16x4 *)(t + i * PLANE + at(row, c16 >> 1) + (c16 & 1) * 8) = h;
            float a = v[0], b = v[1], c = v[2], d = v[3];
            at_less((bf16x2){h[0], h[1]}, a, b);
            at_less((bf16x2){h[2], h[3]}, c, d);
            v = (f32x4){a, b, c, d};
        }
    }
    // acc[db] (32 values of d x 32 columns) += tile[rows base..base+31][d]^T * w, w in the result layout (rows = the tile's rows); FINE:
    // in bf16 w goes in as two parts
    template <bool FINE = false> static __device__ __forceinline__ void acc_t(f32x16 (&acc)[DP / 32], const char *t, int base, const f32x16 &w, int lane)
    {
        const int h = lane >> 5, j = lane & 15, row0 = base + 4 * h + (j >> 2), part = ((lane >> 4) & 1) * 2 + ((j & 3) >> 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x8 x = s ? __builtin_shufflevector(w, w, 8, 9, 10, 11, 12, 13, 14, 15) : __builtin_shufflevector(w, w, 0, 1, 2, 3, 4, 5, 6, 7);
            at_op<T> b;                           // bf16: one rounding to 8 bits (FINE: to 16); the sum stays in 32
            bf16x8 low = (bf16x8)(0.f);
            if (FINE && N == 1) {
                b.p[0] = at_next(x);
                low = __builtin_convertvector(x, bf16x8);
            } else at_cut(x, b);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
                typedef __attribute__((address_space(3))) s16x4 *lp;
                at_op<T> a;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(t + i * PLANE + at(row0 + 16 * s, db * 4 + part) + (j & 1) * 8));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(t + i * PLANE + at(row0 + 16 * s + 8, db * 4 + part) + (j & 1) * 8));
                    a.p[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
                if (FINE && N == 1) acc[db] = at_mfma(a.p[0], low, acc[db]);
                acc[db] = at_mma(a, b, acc[db]);
            }
        }
    }
};

// what a call is made of, on the device's side
template <typename T> struct at_args {
    const T *q, *k, *v, *g;                       // g: gradient of the output (backward)
    T *o, *dk;                                    // o: output / dq; dk, dv
    T *dv, *rest;                                 // rest: what rounding took from the output (bf16; may be NULL)
    float *lse;                                   // forward: output (b, hq, nq)
    const f32x2 *stat;                            // backward: (b, hq, nq) pairs of a row's log-sum in base 2 and -delta
    float *part;                                  // partial results of a split call
    const int32_t *qc, *kc;
    const u32 *bits;                              // pair mask, 32 keys a word: (masks, nq, words)
    int64_t qs[3], ks[3], vs[3], gs[3];           // strides of batch, row, head, in values
    int64_t bs;                                   // words of an image's mask (0: one mask for all)
    int words, batch, nq, nk, hq, hk, d, tiles, splits, per;    // per: rows or keys of a split, a multiple of the tile
    float c, scale, slack;                        // c = scale * log2(e); slack = 8 / c
};

// four values of the output, and what rounding took from them
template <typename T> __device__ __forceinline__ void at_out(const at_args<T> &a, T *o, f32x4 x)
{
    typedef typename at_vec<T>::quad quad;
    const quad r = __builtin_convertvector(x, quad);
    *(quad *)o = r;
    if (sizeof(T) == 2 && a.rest) *(quad *)(a.rest + (o - a.o)) = __builtin_convertvector(x - __builtin_convertvector(r, f32x4), quad);
}

__device__ __forceinline__ int at_count(const int32_t *c, int b, int n) { return c ? min(max(c[b], 0), n) : n; }

// Workgroups go round the eight XCDs.  The tiles of one (image, key head) stay on one XCD, so that they find its keys in one L2, and
// (image, key head) pairs go round the XCDs one by one, so that images of different counts even out; what is left over of a
// multiple of eight pairs is cut into eight runs of tiles.
__device__ __forceinline__ int at_xcd_id(int per)  // per: tiles x splits of a pair -> pair * per + tile
{
    const int x = blockIdx.x & 7, j = blockIdx.x >> 3, pairs = (int)(gridDim.x / per), whole = pairs & ~7;
    if (j < (whole >> 3) * per) return (x + 8 * (j / per)) * per + j % per;
    const int n = (pairs - whole) * per, q = n >> 3, r = n & 7;
    return whole * per + x * q + min(x, r) + j - (whole >> 3) * per;
}

// Images of different counts: the workgroups that come first take the images with the longest walk (keys in the forward and dq
// kernels, rows in the other), so that what runs last is short.  i-th image in that order (equal ones by index); every wave finds it
// for itself from the counts.
__device__ __forceinline__ int at_image(int i, int batch, const int32_t *counts, int n)
{
    if (!counts || batch < 2 || batch > 64) return i;
    const int lane = threadIdx.x & 63, w = lane < batch ? at_count(counts, lane, n) : -1;
    int rank = 0;
    for (int j = 0; j < batch; ++j) {
        const int o = __builtin_amdgcn_readlane(w, j);
        rank += o > w || (o == w && j < lane);
    }
    return __ffsll((unsigned long long)__ballot(lane < batch && rank == i)) - 1;
}

// the word of a row's mask that holds keys kb .. kb + 31 (kb a multiple of 32), without those from k1 on
__device__ __forceinline__ u32 at_word(const u32 *row, int kb, int k1)
{
    if (kb >= k1) return 0;
    const u32 w = row[kb >> 5];
    return k1 - kb < 32 ? w & ((1u << (k1 - kb)) - 1) : w;
}

template <typename T> __device__ __forceinline__ u32x4 at_load_chunk(const T *p) { return *(const u32x4 *)p; }

// A workgroup's loader of row tiles: thread t takes 16 bytes, t % CPR, of rows t / CPR, + STEP, ...  Buffer loads: the tile's address is
// uniform, a lane's offset inside it fixed, and a lane with nothing to load (a row behind the end, a chunk behind d) asks for an
// offset out of range and gets zeros.  A tile spans less than 2^31 bytes (at_aligned).
#define AT_OUT 0x7fffffff
#define AT_VM0 0x0f70                             // s_waitcnt vmcnt(0), the other counters free
template <typename T, int DP, int ROWS, bool LEAN = false> struct at_loader {
    typedef at_tile<T, DP, ROWS> tile;
    static constexpr int CPR = DP * (int)sizeof(T) / 16, STEP = AT_THREADS / CPR, NL = ROWS / STEP > 0 ? ROWS / STEP : 1;
    const T *base;
    int64_t stride;
    int bytes, row0_, c16_, off_;                 // bytes: of a row; off: of the first row's chunk
    __device__ __forceinline__ at_loader(const T *p, int64_t st, int d) : base(p), stride(st), bytes(d * (int)sizeof(T))
    {
        place(threadIdx.x, row0_, c16_, off_);
    }
    __device__ __forceinline__ void place(int t, int &row0, int &c16, int &off) const
    {
        row0 = t / CPR;
        c16 = t % CPR;
        off = c16 * 16 < bytes ? row0 * (int)(stride * (int)sizeof(T)) + c16 * 16 : AT_OUT;
    }
    // LEAN: a thread's place is formed anew in every turn, where keeping it would cost registers that are not there
    __device__ __forceinline__ void place(int &row0, int &c16, int &off) const
    {
        if (LEAN) {
            int t = threadIdx.x;
            asm volatile("" : "+v"(t));
            place(t, row0, c16, off);
        } else { row0 = row0_; c16 = c16_; off = off_; }
    }
    __device__ __forceinline__ void load(u32x4 (&r)[NL], int64_t first, int rows) const
    {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)(base + first * stride), 0, AT_OUT, 0x00027000);
        int row0, c16, off;
        place(row0, c16, off);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int o = row0 + i * STEP < rows ? off : AT_OUT;
            r[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, i * STEP * (int)(stride * (int)sizeof(T)), 0));
        }
    }
    __device__ __forceinline__ void store(char *lds, const u32x4 (&r)[NL]) const
    {
        int row0, c16, off;
        place(row0, c16, off);
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (ROWS >= STEP || row0 < ROWS) tile::put(lds, row0 + i * STEP, c16, r[i]);
    }
};

// with a pair mask, a row of K, V, Q or dO that some rows may not see must not reach them through 0 * NaN: non-finite values
// are put to zero in the staged copy, and the caller marks the row so that those who do see it get NaN.  Values of 32 bits that round to
// infinity as their first part count with them
template <typename T> __device__ __forceinline__ bool at_scrub(u32x4 &x)
{
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 2) {
            const bool lo = (x[i] & 0x7f80u) == 0x7f80u, hi = (x[i] & 0x7f800000u) == 0x7f800000u;
            if (lo) x[i] &= 0xffff0000u;
            if (hi) x[i] &= 0x0000ffffu;
            bad |= lo | hi;
        } else {
            const bool b = (x[i] & 0x7fffffffu) >= 0x7f7f8000u;
            if (b) x[i] = 0;
            bad |= b;
        }
    }
    return bad;
}
#define AT_NAN4 ((u32x4){0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu})   // NaN in bf16 and in fp32

// ------------------------------------------------------------------ forward
// The wave that has scores to multiply goes first, then one that has values to, then the vector work: with equal priorities the two
// waves of a SIMD drift into the same phase and the matrix unit waits (16000 x 128: forward 1101 -> 1040 us, dq 1575 -> 1511, dk, dv
// 2253 -> 2140).  In bf16 up to 64, where three
// or four waves share a SIMD, it only keeps the scheduler from mixing the phases (dk, dv 101 -> 126); in fp32, whose products are six times as
// many, it helps there too (8 x 2000 x 64: forward 375 -> 353, dk, dv 668 -> 643).
#define AT_PRIO(p) do { if (DP == 128 || sizeof(T) == 4) __builtin_amdgcn_s_setprio(p); } while (0)

// Never taken (d is 8 at least): it parts a turn of the loop between the products and the exponentials.  In one piece the scheduler
// keeps so many operands of later products in registers that others are spilled (16001 x 128: dk, dv 2545 -> 2220 us, dq 1650 -> 1530).
#define AT_PART(when) if ((when) && a.d <= 0) break

// Keys of a tile (KT forward, KT_Q dq) and waves of a SIMD that the registers are cut for.  Up to 64 values a head in bf16, four
// waves with tiles of 32 keys hide more than three with 64 (16 x 2000 rows: 174 to 180 us); at 128 two fit, and tiles of 64 halve
// the barriers (forward); dq and (dk, dv) keep more in registers.  The limits also keep matrix results in registers that the
// vector unit can read.
template <typename T, int DP> struct at_shape {
    static constexpr int BYTES = sizeof(T) * DP, H = sizeof(T) == 2;
    static constexpr int KT = H && DP == 128 ? 64 : 32, KT_Q = 32;
    static constexpr int OCC = BYTES > 256 ? 1 : H && DP <= 64 ? 4 : 2, OCC_Q = BYTES > 256 ? 1 : H && DP <= 64 ? 3 : 2, OCC_KV = H ? DP <= 64 ? 3 : 2 : BYTES > 256 ? 1 : 2;
};

// A workgroup: 128 rows (a wave: 32, one per lane pair), all keys of its split in tiles of KT.  K and V tiles are double buffered
// in LDS; the next tile's loads are on their way while this one is computed.  Per 32 x 32 scores a wave spends 8 d / 64 matrix
// instructions of 32 cycles and about 90 vector instructions (scale, exponential, sum, maximum, rounding; the 16 exponentials at a
// quarter of the others' rate).  With 64 values a head the vector unit is busy 67% of the time and the matrix unit 32%, with 128 48%
// and 49%: they take turns, and neither alone is the bound.  Measured, bf16: 16 x 2000 rows and keys, 8 heads of 64: 172 us, 762
// TFLOP/s; 16000, 8 heads of 128: 1050 us, 999 TFLOP/s (a large matrix product reaches 1195); fp32, 8 x 2000, 8 heads of 64: 339 us,
// 193 TFLOP/s (a library's matrix product of 32 bits: 153; by 32-bit matrix instructions it took 590).
template <typename T, int DP, bool MASK>
__global__ __launch_bounds__(AT_THREADS, (at_shape<T, DP>::OCC)) void k_attn_fwd(const at_args<T> a)
{
    constexpr int NG = DP / 16, NB = DP / 32, KT = at_shape<T, DP>::KT, U = KT / 32;
    typedef at_tile<T, DP, KT> tile;
    __shared__ __attribute__((aligned(16))) char lds[2][2][tile::BYTES];

    const int id = at_xcd_id(a.tiles * a.splits), tix = id % a.tiles, sp = (id / a.tiles) % a.splits, bh = id / a.tiles / a.splits;
    const int b = at_image(bh / a.hk, a.batch, a.kc, a.nk), hk = bh % a.hk, G = a.hq / a.hk;
    const int nq = at_count(a.qc, b, a.nq), nk = at_count(a.kc, b, a.nk);
    const int R = G * nq, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;

    if (sp == 0) {                                // rows behind the image's last one: nothing seen
        const int pad = a.nq - nq;
        for (int p = tix; p < G * pad; p += a.tiles) {
            const int hq = hk * G + p / pad, n = nq + p % pad;
            T *o = a.o + (((int64_t)b * a.nq + n) * a.hq + hq) * a.d;
            for (int d = threadIdx.x; d < a.d; d += AT_THREADS) {
                o[d] = (T)0.f;
                if (sizeof(T) == 2 && a.rest) a.rest[o - a.o + d] = (T)0.f;
            }
            if (threadIdx.x == 0) a.lse[((int64_t)b * a.hq + hq) * a.nq + n] = -INFINITY;
        }
    }
    if (tix * 32 * AT_WAVES >= R) return;

    const int r = (tix * AT_WAVES + wave) * 32 + (lane & 31);
    const bool live = r < R;
    const int gh = live ? r / nq : 0, n = live ? r % nq : 0, hq = hk * G + gh;
    const T *qp = a.q + b * a.qs[0] + n * a.qs[1] + hq * a.qs[2];
    at_op<T> qf[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int d = (2 * g + h) * 8;
        at_read(qp + d, live && d < a.d, qf[g]);
    }
    const u32 *mp = MASK ? a.bits + b * a.bs + (int64_t)n * a.words : nullptr;

    const int k0 = sp * a.per, k1 = min(nk, k0 + a.per);
    const at_loader<T, DP, KT> kl(a.k + b * a.ks[0] + hk * a.ks[2], a.ks[1], a.d), vl(a.v + b * a.vs[0] + hk * a.vs[2], a.vs[1], a.d);
    u32x4 kr[kl.NL], vr[kl.NL];
    auto load = [&](int kb) {
        kl.load(kr, kb, k1 - kb);
        vl.load(vr, kb, k1 - kb);
    };
    auto store = [&](int buf) {
        if (MASK) {
#pragma unroll
            for (int i = 0; i < kl.NL; ++i)
                if (at_scrub<T>(vr[i])) kr[i] = AT_NAN4;    // scores of that key become NaN for the rows that see it
        }
        kl.store(lds[buf][0], kr);
        vl.store(lds[buf][1], vr);
    };

    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = (f32x16)(0.f);
    float m = -INFINITY, l = 0.f;                 // maximum in use (of s / scale, at most slack below the true one), this lane's part of the sum
    float lost = 0.f;                             // what rounding added to l: see the end of a turn

    u32 mw[U], mnext[U];                          // MASK: this tile's words and the next one's
    if (k0 < k1) {
        load(k0);
        store(0);
#pragma unroll
        for (int u = 0; u < U; ++u) mw[u] = MASK ? at_word(mp, k0 + 32 * u, k1) : 0;
    }
    __builtin_amdgcn_s_waitcnt(AT_VM0);           // what the loop keeps in registers has arrived: no turn of it waits for a load but its own
    __syncthreads();
    int buf = 0;
    for (int kb = k0; kb < k1; kb += KT, buf ^= 1) {
        const bool more = kb + KT < k1;
        if (more) load(kb + KT);
#pragma unroll
        for (int u = 0; u < U; ++u) mnext[u] = MASK ? at_word(mp, kb + KT + 32 * u, k1) : 0;
        const char *K = lds[buf][0], *V = lds[buf][1];
        f32x16 s[U];
        AT_PRIO(2);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = (f32x16)(0.f);
#pragma unroll
            for (int g = 0; g < NG; ++g) s[u] = at_mma(tile::row(K, u * 32 + (lane & 31), 2 * g + h), qf[g], s[u]);
        }
        AT_PRIO(0);
        if (MASK || !more) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int left = k1 - kb - u * 32;
                const u32 w = (MASK ? mw[u] : left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[u][e] = w & (1u << (8 * (e >> 2) + (e & 3))) ? s[u][e] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int e = 1; e < 16 * U; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
        float mx2;
        at_both(mx, mx, mx2);
        const float mn = fmaxf(m, fmaxf(mx, mx2));
        if (__any(mn > m + a.slack)) {            // otherwise the old maximum still does: no p exceeds 2^8
            const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
            l *= al;
            lost *= al;
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= al;
            m = mn;
        }
        AT_PART(DP == 128);
        const float base = m == -INFINITY ? 0.f : m * a.c;
        f32x4 sum;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[u][e], a.c, -base));
                s[u][e] = p;
                sum[e & 3] = u == 0 && e < 4 ? p : sum[e & 3] + p;
            }
            AT_PRIO(1);
            tile::acc_t(o, V, u * 32, s[u], lane);
            AT_PRIO(0);
        }
        // A long walk over keys of like scores adds thousands of like values, whose roundings all point one way: a tile's are summed first,
        // and what rounding did to l is taken from the next tile's sum (one by one: 7e-5 of l after 16000 keys, by tiles alone 6e-6, so 4e-8)
        const float x = ((sum[0] + sum[1]) + (sum[2] + sum[3])) - lost, y = l + x;
        lost = (y - l) - x;
        l = y;
        if (more) store(buf ^ 1);
#pragma unroll
        for (int u = 0; u < U; ++u) mw[u] = mnext[u];
        __syncthreads();
    }
    float l2;
    at_both(l, l, l2);
    l += l2;
    if (!live) return;
    const bool none = m == -INFINITY && !(l != l);
    const float inv = none ? 0.f : 1.f / l;
    const float lse2 = none ? -INFINITY : fmaf(m, a.c, __builtin_amdgcn_logf(l));
    if (a.splits > 1) {
        // partial result of the split: normalised values and their log-sum, joined by k_attn_join
        const int64_t row = ((int64_t)b * a.hq + hq) * a.nq + n, rows = (int64_t)(gridDim.x / a.tiles / a.splits) * G * a.nq;
        float *po = a.part + rows * a.splits + (row * a.splits + sp) * a.d;
        if (h == 0) a.part[row * a.splits + sp] = lse2;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = i * 32 + 2 * e + 4 * h;
                if (d < a.d) *(f32x4 *)(po + d) = (f32x4){o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv};
            }
        return;
    }
    T *op = a.o + (((int64_t)b * a.nq + n) * a.hq + hq) * a.d;
    if (h == 0) a.lse[((int64_t)b * a.hq + hq) * a.nq + n] = lse2 * AT_LN2;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = i * 32 + 2 * e + 4 * h;
            if (d < a.d) at_out(a, op + d, (f32x4){o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv});
        }
}

// Joins the splits of a row by their log-sums, four values of d a thread.  Up to 16 splits (MANY false) a row has 32 threads, eight
// rows a workgroup; with more (few rows, a long walk) a workgroup has 32 values of one row, and its 32 groups of eight threads deal
// the splits among themselves and add up through LDS (126 splits of 16 rows: 68 us by a wave a row, 11 by a workgroup a row, 7 so).
#define AT_JOIN_FEW 16
template <typename T, bool MANY>
__global__ __launch_bounds__(AT_THREADS) void k_attn_join(const at_args<T> a, int64_t rows)
{
    constexpr int LANES = MANY ? 8 : 32, GROUPS = AT_THREADS / LANES;
    __shared__ __attribute__((aligned(16))) f32x4 red[MANY ? GROUPS : 1][LANES];
    __shared__ float tots[GROUPS], tops[AT_WAVES];
    const int grp = threadIdx.x / LANES, sub = threadIdx.x % LANES, cuts = MANY ? (a.d + 31) / 32 : 1;
    const int64_t row = MANY ? blockIdx.x / cuts : (int64_t)blockIdx.x * GROUPS + grp;
    const int d = (MANY ? (int)(blockIdx.x % cuts) * 32 : 0) + sub * 4;
    if (row >= rows) return;                      // MANY: the whole workgroup
    const u32 bh = (u32)row / a.nq, b = bh / a.hq;
    const int n = (int)((u32)row - bh * a.nq), hq = (int)(bh - b * a.hq);
    if (n >= at_count(a.qc, b, a.nq)) return;     // written by the first kernel
    const float *ls = a.part + row * a.splits, *po = a.part + rows * a.splits + row * a.splits * a.d + d;
    float m = -INFINITY;
    for (int s = MANY ? (int)threadIdx.x : sub; s < a.splits; s += MANY ? AT_THREADS : LANES) m = fmaxf(m, ls[s]);
#pragma unroll
    for (int x = MANY ? 32 : LANES / 2; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
    if (MANY) {
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < AT_WAVES; ++w) m = fmaxf(m, tops[w]);
    }
    const float base = m == -INFINITY ? 0.f : m;
    const bool in = d < a.d;
    float tot = 0.f;
    f32x4 v = (f32x4)(0.f);
#pragma unroll 4
    for (int s = MANY ? grp : 0; s < a.splits; s += MANY ? GROUPS : 1) {
        const float w = __builtin_amdgcn_exp2f(ls[s] - base);
        tot += w;
        if (in) v += *(const f32x4 *)(po + (int64_t)s * a.d) * w;
    }
    if (MANY) {
        red[grp][sub] = v;
        if (sub == 0) tots[grp] = tot;
        __syncthreads();
        if (grp) return;
        for (int g = 1; g < GROUPS; ++g) {
            v += red[g][sub];
            tot += tots[g];
        }
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
    if (in) at_out(a, a.o + (((int64_t)b * a.nq + n) * a.hq + hq) * a.d + d, v * inv);
    if (d == 0) a.lse[row] = tot == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(tot)) * AT_LN2;
}

// ------------------------------------------------------------------ backward
// How ds enters its products in bf16.  The sum of ds over a row's keys is 0, so dq and dk are what is left of larger terms, the more so
// the fewer keys a row sees.  In images of up to AT_FEW keys (and under a pair mask, which may leave few) ds goes in as two parts, 16 bits;
// elsewhere one rounding to 8 bits is of no more weight than that of the result.  AT_COUNTED: each image's count decides, whatever the
// padded size: the kernel holds both walks, whole, so that neither's registers bind the other's.
enum { AT_PLAIN, AT_FINE, AT_COUNTED, AT_MASKED };
#define AT_FEW 512
#define AT_CUT(nk) (MODE == AT_COUNTED ? (nk) <= AT_FEW : MODE != AT_PLAIN)
// delta_i = do_i . o_i and the rows' log-sums in base 2; a row that sees nothing gets +inf there, so that its p is 0.  From the output as
// rounded to bf16 alone delta would be off by 2^-8 of its terms, which where few keys are seen is as much as ds itself (one key: ds is 0);
// with what rounding took, by 2^-16.  Bound by memory: 8 images of 1000 to 2000 rows x 8 x 64 bf16: 11 us, 3.6 TB/s.
template <typename T, bool MASK>
__global__ __launch_bounds__(AT_THREADS) void k_attn_delta(const at_args<T> a, const T *__restrict__ out, const float *__restrict__ lse, f32x2 *__restrict__ stat,
                                                           u32 rows)
{
    constexpr int CH = 16 / (int)sizeof(T), LPR = 128 / CH, RPB = AT_THREADS / LPR;
    const int sub = threadIdx.x % LPR;
    const u32 row = blockIdx.x * RPB + threadIdx.x / LPR;     // (b, n, hq), heads innermost as in memory; fewer than 2^28 (at_check)
    if (row >= rows) return;
    const u32 bn = row / a.hq, b = bn / a.nq;
    const int hq = (int)(row - bn * a.hq), n = (int)(bn - b * a.nq);
    const int64_t at = ((int64_t)b * a.hq + hq) * a.nq + n;
    const bool live = n < at_count(a.qc, b, a.nq);
    float sum = 0.f;
    int bad = 0;
    const int d = sub * CH;
    if (live && d < a.d) {
        const typename at_vec<T>::frag x = *(const typename at_vec<T>::frag *)(a.g + b * a.gs[0] + n * a.gs[1] + hq * a.gs[2] + d);
        const typename at_vec<T>::frag y = *(const typename at_vec<T>::frag *)(out + (int64_t)row * a.d + d);
#pragma unroll
        for (int i = 0; i < CH; ++i) sum = fmaf((float)x[i], (float)y[i], sum);
        if (sizeof(T) == 2 && a.rest) {
            const typename at_vec<T>::frag z = *(const typename at_vec<T>::frag *)(a.rest + (int64_t)row * a.d + d);
#pragma unroll
            for (int i = 0; i < CH; ++i) sum = fmaf((float)x[i], (float)z[i], sum);
        }
        if (MASK) {
            u32x4 xs = __builtin_bit_cast(u32x4, x), qs = at_load_chunk(a.q + b * a.qs[0] + n * a.qs[1] + hq * a.qs[2] + d);
            bad = (int)at_scrub<T>(xs) | (int)at_scrub<T>(qs);
        }
    }
#pragma unroll
    for (int x = LPR / 2; x; x >>= 1) {
        sum += __shfl_xor(sum, x, 64);
        if (MASK) bad |= __shfl_xor(bad, x, 64);
    }
    if (sub) return;
    const float l = live ? lse[at] : -INFINITY;
    stat[at] = (f32x2){bad ? __builtin_nanf("") : l == -INFINITY ? INFINITY : l * AT_LOG2E, -sum};
}

// dq: a workgroup owns 128 rows and walks the keys as the forward does; K is read as rows (scores) and transposed (dq), V as rows (dp).
// Three products a tile.  Measured, bf16: 16 x 2000, 8 heads of 64: 247 us, 796 TFLOP/s; 16000, 8 heads of 128: 1491 us, 1055 TFLOP/s;
// fp32, 8 x 2000, 8 heads of 64: 464 us, 212 TFLOP/s (by 32-bit matrix instructions 810).  About 120 vector instructions a tile, of which
// some 45 select by the keys' end, which only the last tile needs; busy 57% of the time at 64, the matrix unit 33%.
template <typename T, int DP, int MODE>
__global__ __launch_bounds__(AT_THREADS, (at_shape<T, DP>::OCC_Q)) void k_attn_dq(const at_args<T> a)
{
    constexpr bool MASK = MODE == AT_MASKED;
    typedef typename at_vec<T>::quad quad;
    constexpr int NG = DP / 16, NB = DP / 32, KT = at_shape<T, DP>::KT_Q, U = KT / 32;
    typedef at_tile<T, DP, KT> tile;
    __shared__ __attribute__((aligned(16))) char lds[2][2][tile::BYTES];

    const int id = at_xcd_id(a.tiles * a.splits), tix = id % a.tiles, sp = (id / a.tiles) % a.splits, bh = id / a.tiles / a.splits;
    const int b = at_image(bh / a.hk, a.batch, a.kc, a.nk), hk = bh % a.hk, G = a.hq / a.hk;
    const int nq = at_count(a.qc, b, a.nq), nk = at_count(a.kc, b, a.nk);
    const int R = G * nq, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;

    if (sp == 0) {
        const int pad = a.nq - nq;
        for (int p = tix; p < G * pad; p += a.tiles) {
            T *o = a.o + (((int64_t)b * a.nq + nq + p % pad) * a.hq + hk * G + p / pad) * a.d;
            for (int d = threadIdx.x; d < a.d; d += AT_THREADS) o[d] = (T)0.f;
        }
    }
    if (tix * 32 * AT_WAVES >= R) return;

    const int r = (tix * AT_WAVES + wave) * 32 + (lane & 31);
    const bool live = r < R;
    const int gh = live ? r / nq : 0, n = live ? r % nq : 0, hq = hk * G + gh;
    auto walk = [&](auto cut) {                   // cut: ds goes in as two parts
        const T *qp = a.q + b * a.qs[0] + n * a.qs[1] + hq * a.qs[2], *gp = a.g + b * a.gs[0] + n * a.gs[1] + hq * a.gs[2];
        at_op<T> qf[NG], gf[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int d = (2 * g + h) * 8;
            at_read(qp + d, live && d < a.d, qf[g]);
            at_read(gp + d, live && d < a.d, gf[g]);
        }
        const int64_t at = ((int64_t)b * a.hq + hq) * a.nq + n;
        const f32x2 stat = live ? a.stat[at] : (f32x2){INFINITY, 0.f};
        const float lse2 = stat[0];
        const u32 *mp = MASK ? a.bits + b * a.bs + (int64_t)n * a.words : nullptr;

        const int k0 = sp * a.per, k1 = min(nk, k0 + a.per);
        const at_loader<T, DP, KT> kl(a.k + b * a.ks[0] + hk * a.ks[2], a.ks[1], a.d), vl(a.v + b * a.vs[0] + hk * a.vs[2], a.vs[1], a.d);
        u32x4 kr[kl.NL], vr[kl.NL];
        auto load = [&](int kb) {
            kl.load(kr, kb, k1 - kb);
            vl.load(vr, kb, k1 - kb);
        };
        auto store = [&](int buf) {
            if (MASK) {
#pragma unroll
                for (int i = 0; i < kl.NL; ++i)
                    if (at_scrub<T>(kr[i])) vr[i] = AT_NAN4;    // dp of that key becomes NaN
            }
            kl.store(lds[buf][0], kr);
            vl.store(lds[buf][1], vr);
        };

        f32x16 o[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) o[i] = (f32x16)(0.f);
        u32 mw[U], mnext[U];                          // MASK: this tile's words and the next one's
        if (k0 < k1) {
            load(k0);
            store(0);
#pragma unroll
            for (int u = 0; u < U; ++u) mw[u] = MASK ? at_word(mp, k0 + 32 * u, k1) : 0;
        }
        __builtin_amdgcn_s_waitcnt(AT_VM0);           // what the loop keeps in registers has arrived: no turn of it waits for a load but its own
        __syncthreads();
        int buf = 0;
        for (int kb = k0; kb < k1; kb += KT, buf ^= 1) {
            const bool more = kb + KT < k1;
            if (more) load(kb + KT);
#pragma unroll
            for (int u = 0; u < U; ++u) mnext[u] = MASK ? at_word(mp, kb + KT + 32 * u, k1) : 0;
            const char *K = lds[buf][0], *V = lds[buf][1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                f32x16 s = (f32x16)(0.f), dp = (f32x16)(stat[1]);
                AT_PRIO(2);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    s = at_mma(tile::row(K, u * 32 + (lane & 31), 2 * g + h), qf[g], s);
                    dp = at_mma(tile::row(V, u * 32 + (lane & 31), 2 * g + h), gf[g], dp);
                }
                AT_PRIO(0);
                const int left = k1 - kb - u * 32;
                const u32 w = (MASK ? mw[u] : left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u) >> (4 * h);
                AT_PART(DP == 128);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float ds = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -lse2)) * dp[e];
                    if (MASK || !more) ds = w & (1u << (8 * (e >> 2) + (e & 3))) ? ds : 0.f;
                    s[e] = ds;
                }
                AT_PRIO(1);
                tile::template acc_t<decltype(cut)::value>(o, K, u * 32, s, lane);
                AT_PRIO(0);
            }
            if (more) store(buf ^ 1);
#pragma unroll
            for (int u = 0; u < U; ++u) mw[u] = mnext[u];
            __syncthreads();
        }
        if (!live) return;
        float *po = a.part + (((int64_t)b * a.hq + hq) * a.nq + n) * a.splits * a.d + (int64_t)sp * a.d;
        T *op = a.o + (((int64_t)b * a.nq + n) * a.hq + hq) * a.d;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = i * 32 + 2 * e + 4 * h;
                const f32x4 x = (f32x4){o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]} * a.scale;
                if (d >= a.d) continue;
                if (a.splits > 1) *(f32x4 *)(po + d) = x;
                else *(quad *)(op + d) = __builtin_convertvector(x, quad);
            }
    };
    if (AT_CUT(nk)) walk(std::true_type());
    else walk(std::false_type());
}

#define AT_RT 32
// dk, dv: a workgroup owns 128 keys (a wave: 32, one per lane pair) and walks the rows; Q and dO tiles are read as rows (scores,
// dp) and transposed (dk, dv).  Four products a tile, and 2 x 32 x d accumulators a wave, which bound how many waves share a SIMD.
// Measured, bf16: 16 x 2000, 8 heads of 64: 359 us, 730 TFLOP/s; 16000, 8 heads of 128: 2135 us, 982 TFLOP/s; fp32, 8 x 2000, 8 heads of
// 64: 614 us, 213 TFLOP/s (by 32-bit matrix instructions 1084).  About 150 vector instructions a tile at 64, half of them addresses.
template <typename T, int DP, int MODE>
__global__ __launch_bounds__(AT_THREADS, (MODE == AT_MASKED && at_shape<T, DP>::OCC_KV == 3 ? 2 : at_shape<T, DP>::OCC_KV)) void k_attn_dkv(const at_args<T> a)
{
    constexpr bool MASK = MODE == AT_MASKED;
    typedef typename at_vec<T>::quad quad;
    constexpr int NG = DP / 16, NB = DP / 32, KT = AT_RT;
    typedef at_tile<T, DP, KT> tile;
    __shared__ __attribute__((aligned(16))) char lds[2][2][tile::BYTES];
    __shared__ __attribute__((aligned(16))) float st[2][2][KT];
    constexpr bool LEAN = sizeof(T) == 2 && DP >= 64;
    constexpr bool VL = sizeof(T) == 2 && DP == 128;          // V stays in LDS: its registers are what would keep a second wave off the SIMD
    __shared__ __attribute__((aligned(16))) char vt[VL ? 32 * AT_WAVES * tile::RB : 16];
    __shared__ __attribute__((aligned(16))) u32 mws[2][AT_WAVES][MASK ? KT : 4];

    const int id = at_xcd_id(a.tiles * a.splits), tix = id % a.tiles, sp = (id / a.tiles) % a.splits, bh = id / a.tiles / a.splits;
    const int b = at_image(bh / a.hk, a.batch, a.qc, a.nq), hk = bh % a.hk, G = a.hq / a.hk;
    const int nq = at_count(a.qc, b, a.nq), nk = at_count(a.kc, b, a.nk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    // the walk: row tiles of each query head of the group in turn; none where all keys lie behind the image's last one (zeros)
    const int ht = (nq + KT - 1) / KT, W = tix * 32 * AT_WAVES < nk ? G * ht : 0;
    const int key = (tix * AT_WAVES + wave) * 32 + (lane & 31);
    const bool live = key < nk;

    auto walk = [&](auto cut) {                   // cut: ds goes in as two parts
        const T *kp = a.k + b * a.ks[0] + (live ? key : 0) * a.ks[1] + hk * a.ks[2], *vp = a.v + b * a.vs[0] + (live ? key : 0) * a.vs[1] + hk * a.vs[2];
        at_op<T> kf[NG], vf[VL ? 1 : NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int d = (2 * g + h) * 8;
            at_op<T> x;
            at_read(kp + d, live && d < a.d, kf[g]);
            at_read(vp + d, live && d < a.d, x);
            if (VL) *(at_op<T> *)(vt + (wave * NG + g) * 1024 + lane * 16) = x;
            else vf[VL ? 0 : g] = x;
        }

        const int w0 = min(W, sp * a.per), w1 = min(W, w0 + a.per);
        int wg = ht ? w0 / ht : 0, wn = ht ? w0 - wg * ht : 0;       // the next tile to load
        u32x4 qr[at_loader<T, DP, KT, LEAN>::NL], gr[at_loader<T, DP, KT, LEAN>::NL];
        const at_loader<T, DP, KT, LEAN> ql(a.q + b * a.qs[0] + hk * G * a.qs[2], a.qs[1], a.d), gl(a.g + b * a.gs[0] + hk * G * a.gs[2], a.gs[1], a.d);
        const u32 *mp = MASK ? a.bits + b * a.bs : nullptr;
        u64 sr = 0;
        u32 mr = 0;
        auto load = [&]() {
            const int n0 = wn * KT, rows = nq - n0;
            at_loader<T, DP, KT, LEAN> q1 = ql, g1 = gl;
            q1.base += wg * a.qs[2];
            g1.base += wg * a.gs[2];
            q1.load(qr, n0, rows);
            g1.load(gr, n0, rows);
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)(a.stat + ((int64_t)b * a.hq + hk * G + wg) * a.nq + n0), 0, AT_OUT, 0x00027000);
            // the rows' statistics; zeros behind the end, where q and grad_out are zeros too
            sr = __builtin_bit_cast(u64, __builtin_amdgcn_raw_buffer_load_b64(rs, (int)threadIdx.x < min(KT, rows) ? (int)threadIdx.x * 8 : AT_OUT, 0, 0));
            if (MASK && threadIdx.x < KT * AT_WAVES) {   // the words of the tile's rows for each wave's keys
                const int n = threadIdx.x / AT_WAVES, kw = tix * AT_WAVES + threadIdx.x % AT_WAVES;
                mr = n < rows && kw < a.words ? mp[(int64_t)(n0 + n) * a.words + kw] : 0;
            }
            if (++wn == ht) { wn = 0; ++wg; }
        };
        auto store = [&](int buf) {
            if (MASK) {                               // the row's log-sum already says NaN (k_attn_delta)
#pragma unroll
                for (int i = 0; i < ql.NL; ++i) {
                    at_scrub<T>(qr[i]);
                    at_scrub<T>(gr[i]);
                }
            }
            ql.store(lds[buf][0], qr);
            gl.store(lds[buf][1], gr);
            if (MASK && threadIdx.x < KT * AT_WAVES) mws[buf][threadIdx.x % AT_WAVES][threadIdx.x / AT_WAVES] = mr;
            if (threadIdx.x < KT) {
                st[buf][0][threadIdx.x] = __builtin_bit_cast(f32x2, sr)[0];
                st[buf][1][threadIdx.x] = __builtin_bit_cast(f32x2, sr)[1];
            }
        };

        f32x16 ok[NB], ov[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) ok[i] = ov[i] = (f32x16)(0.f);
        if (w0 < w1) {
            load();
            store(0);
        }
        __builtin_amdgcn_s_waitcnt(AT_VM0);           // what the loop keeps in registers has arrived: no turn of it waits for a load but its own
        __syncthreads();
        int buf = 0;
        for (int w = w0; w < w1; ++w, buf ^= 1) {
            const bool more = w + 1 < w1;
            if (more) load();
            const char *Q = lds[buf][0], *GO = lds[buf][1];
            // the LDS addresses of a tile are formed anew in every turn: kept across the loop they would cost a wave of the SIMD
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const int lr = ln & 31, lh = ln >> 5;
            f32x16 s = (f32x16)(0.f), dp;
            AT_PRIO(2);
#pragma unroll
            for (int g = 0; g < NG; ++g) s = at_mma(tile::row(Q, lr, 2 * g + lh), kf[g], s);
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = (*(const f32x4 *)&st[buf][1][2 * (e & ~3) + 4 * lh])[e & 3];
#pragma unroll
            for (int g = 0; g < NG; ++g)
                dp = at_mma(tile::row(GO, lr, 2 * g + lh), VL ? *(const at_op<T> *)(vt + (wave * NG + g) * 1024 + ln * 16) : vf[VL ? 0 : g], dp);
            AT_PRIO(0);
            AT_PART(DP >= 64);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -(*(const f32x4 *)&st[buf][0][2 * (e & ~3) + 4 * lh])[e & 3]));
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float ds = s[e] * dp[e];
                if (MASK) {
                    const bool see = live && ((*(const u32x4 *)&mws[buf][wave][2 * (e & ~3) + 4 * lh])[e & 3] >> lr) & 1;
                    s[e] = see ? s[e] : 0.f;
                    ds = see ? ds : 0.f;
                }
                dp[e] = ds;
            }
            AT_PRIO(1);
            tile::acc_t(ov, GO, 0, s, ln);
            tile::template acc_t<decltype(cut)::value>(ok, Q, 0, dp, ln);
            AT_PRIO(0);
            if (more) store(buf ^ 1);
            __syncthreads();
        }
        if (key >= a.nk) return;
        const int64_t rows = (int64_t)(gridDim.x / a.tiles / a.splits) * a.nk, prow = ((int64_t)b * a.hk + hk) * a.nk + key;
        float *pk = a.part + prow * a.splits * a.d + (int64_t)sp * a.d, *pv = pk + rows * a.splits * a.d;
        const int64_t orow = (((int64_t)b * a.nk + key) * a.hk + hk) * a.d;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = i * 32 + 2 * e + 4 * h;
                if (d >= a.d) continue;
                f32x4 x = (f32x4){ok[i][e], ok[i][e + 1], ok[i][e + 2], ok[i][e + 3]} * a.scale, y = (f32x4){ov[i][e], ov[i][e + 1], ov[i][e + 2], ov[i][e + 3]};
                if (!live) x = y = (f32x4)(0.f);
                if (a.splits > 1) {
                    *(f32x4 *)(pk + d) = x;
                    *(f32x4 *)(pv + d) = y;
                } else {
                    *(quad *)(a.dk + orow + d) = __builtin_convertvector(x, quad);
                    *(quad *)(a.dv + orow + d) = __builtin_convertvector(y, quad);
                }
            }
    };
    if (AT_CUT(nk)) walk(std::true_type());
    else walk(std::false_type());
}

// sums a gradient's splits in their order: rows (b, h, n) of the partial sums -> (b, n, h); rows behind a count are left alone; a second
// gradient of the same shape (dv) follows the first one's partial sums
template <typename T>
__global__ __launch_bounds__(AT_THREADS) void k_attn_sum(const float *__restrict__ part, T *__restrict__ out, T *__restrict__ out2, const int32_t *__restrict__ counts, int64_t rows, int heads,
                                                         int nmax, int d, int splits)
{
    typedef typename at_vec<T>::quad quad;
    const u32 i = blockIdx.x * AT_THREADS + threadIdx.x, row = i / (u32)(d / 4);     // a split call has few rows
    if (row >= rows) return;
    const u32 bh = row / nmax, b = bh / heads;
    const int x = (int)(i - row * (d / 4)) * 4, n = (int)(row - bh * nmax), hh = (int)(bh - b * heads);
    if (n >= at_count(counts, b, nmax)) return;
    const float *p = part + ((blockIdx.y ? rows : 0) + (int64_t)row) * splits * d + x;
    f32x4 v = (f32x4)(0.f);
#pragma unroll 4
    for (int s = 0; s < splits; ++s) v += *(const f32x4 *)(p + (int64_t)s * d);
    *(quad *)((blockIdx.y ? out2 : out) + (((int64_t)b * nmax + n) * heads + hh) * d + x) = __builtin_convertvector(v, quad);
}

// pair mask -> bits, once for all heads and passes over it (4 x 509 x 509: the bytes read by every lane for itself cost the three
// kernels 47, 53 and 71 us, the bits 38, 44 and 59; 4 to make them).  A workgroup has 1024 keys of a row, a wave 256: a byte a lane, a ballot for 64.
__global__ __launch_bounds__(AT_THREADS) void k_attn_bits(const uint8_t *__restrict__ mask, int64_t sb, int64_t sr, u32 *__restrict__ bits, u32 blocks, int nq, int nk, int words)
{
    const u32 id = dg_block(), cuts = (nk + 1023) / 1024, r = id / cuts;
    if (id >= blocks) return;
    const int lane = threadIdx.x & 63, k0 = (int)(id - r * cuts) * 1024 + (int)(threadIdx.x >> 6) * 256;
    const uint8_t *m = mask + (int64_t)(r / nq) * sb + (int64_t)(r % nq) * sr;
    uint8_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = k0 + 64 * j + lane;
        v[j] = k < nk ? m[k] : 0;
    }
    u32 x = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const u64 w = __ballot(v[j] != 0);
        if (lane >> 1 == j) x = (u32)(w >> (32 * (lane & 1)));
    }
    const int w = (k0 >> 5) + lane;
    if (lane < 8 && w < words) bits[(int64_t)r * words + w] = x;
}

// ------------------------------------------------------------------ host
// A call that has too few tiles to fill the chip is split along the axis it walks: enough splits for two workgroups on each of
// the 256 CUs, of 128 steps of that axis or more (a multiple of 64); the last one takes what is left, a single step at the least.
static void at_split(int64_t blocks, int64_t walk, int64_t *splits, int64_t *per)
{
    int64_t s = 1;
    if (blocks < 256) s = dg_cdiv(512, blocks > 0 ? blocks : 1);
    const int64_t most = dg_cdiv(walk, 128);
    if (s > most) s = most;
    if (s < 1) s = 1;
    *per = dg_round_up(dg_cdiv(walk > 0 ? walk : 1, s), 64);
    *splits = dg_cdiv(walk > 0 ? walk : 1, *per);
}

struct at_plan { int64_t words, bits, qtiles, ktiles, qsplits, qper, ksplits, kper, rows, stats, qpart, kpart; };

static at_plan at_plan_of(const dg_attn_shape *s)
{
    at_plan p;
    const int64_t g = s->q_heads / s->k_heads, bh = s->batch * s->k_heads;
    p.qtiles = dg_cdiv(g * s->nq, 32 * AT_WAVES);
    p.ktiles = dg_cdiv(s->nk, 32 * AT_WAVES);
    at_split(bh * p.qtiles, s->nk, &p.qsplits, &p.qper);
    at_split(bh * p.ktiles, g * dg_cdiv(s->nq, AT_RT) * AT_RT, &p.ksplits, &p.kper);
    p.kper /= AT_RT;                              // in row tiles
    p.rows = s->batch * s->q_heads * s->nq;
    p.words = dg_cdiv(s->nk, 32);
    p.bits = dg_round_up(s->masks * s->nq * p.words * 4, 256);
    p.stats = dg_round_up(p.rows * 8, 256);
    p.qpart = p.qsplits > 1 ? p.rows * p.qsplits * s->d * 4 : 0;
    p.kpart = p.ksplits > 1 ? 2 * s->batch * s->k_heads * s->nk * p.ksplits * s->d * 4 : 0;
    return p;
}

static int at_check(const dg_attn_shape *s, const char *who)
{
    DG_REQUIRE(s, "%s: null shape", who);
    DG_REQUIRE(s->dtype == DG_F32 || s->dtype == DG_BF16, "%s: type must be DG_F32 or DG_BF16", who);
    DG_REQUIRE(s->batch >= 0 && s->nq >= 0 && s->nk >= 0, "%s: negative size", who);
    DG_REQUIRE(s->k_heads >= 1 && s->q_heads >= 1 && s->q_heads % s->k_heads == 0, "%s: q_heads must be a positive multiple of k_heads", who);
    DG_REQUIRE(s->d >= 8 && s->d <= 128 && s->d % 8 == 0, "%s: head size %lld is not a multiple of 8 from 8 to 128", who, (long long)s->d);
    DG_REQUIRE(s->scale > 0.f && s->scale <= 1e30f, "%s: scale must be positive and at most 1e30", who);
    DG_REQUIRE(s->masks == 0 || s->masks == 1 || s->masks == s->batch, "%s: masks is 0, 1 (for all images) or the batch", who);
    const int64_t most = 1ll << 28;
    DG_REQUIRE(s->batch <= most && s->nk <= most && s->q_heads <= most && s->nq <= most && s->nq * (s->q_heads / s->k_heads) <= most &&
                   s->batch * s->q_heads <= most, "%s: more than 2^28 rows or keys", who);
    const at_plan p = at_plan_of(s);
    const int64_t blocks = (1ll << 32) / AT_THREADS;         // a launch holds fewer than 2^32 threads
    DG_REQUIRE(s->batch * s->k_heads * p.qtiles * p.qsplits < blocks && s->batch * s->k_heads * p.ktiles * p.ksplits < blocks &&
                   dg_cdiv(p.rows, 8) < blocks && s->masks * s->nq * dg_cdiv(s->nk, 1024) < (1ll << 31), "%s: too many tiles for one launch", who);
    return DG_OK;
}

// 16-byte loads: the pointer and every stride that a call steps along; 64 rows of a tile span less than 2^31 bytes
#define AT_ROW_MOST (1ll << 22)
static bool at_aligned(const void *p, const int64_t *st, const dg_attn_shape *s, int64_t n, int64_t heads)
{
    const int64_t e = s->dtype == DG_F32 ? 4 : 2, dims[3] = {s->batch, n, heads};
    if (((uintptr_t)p) & 15) return false;
    for (int i = 0; i < 3; ++i)
        if (dims[i] > 1 && (st[i] < 0 || st[i] * e % 16 || (i == 1 && st[i] > AT_ROW_MOST))) return false;
    return true;
}

extern "C" size_t dg_roi_attn_workspace_bytes(const dg_attn_shape *s, int backward)
{
    if (at_check(s, "roi_attn") != DG_OK) return 0;
    const at_plan p = at_plan_of(s);
    if (!backward) return (size_t)(p.bits + (p.qpart ? p.qpart + p.rows * p.qsplits * 4 : 0));
    return (size_t)(p.bits + p.stats + (p.qpart > p.kpart ? p.qpart : p.kpart));
}

template <typename T>
static at_args<T> at_fill(const dg_attn_shape *s, const void *q, const void *k, const void *v, const int32_t *qc, const int32_t *kc)
{
    at_args<T> a = {};
    a.q = (const T *)q; a.k = (const T *)k; a.v = (const T *)v;
    a.qc = qc; a.kc = kc;
    // an axis of one has no stride: whatever the caller's is, it would enter the loaders' 32-bit offsets of rows that are not there
    const int64_t qn[3] = {s->batch, s->nq, s->q_heads}, kn[3] = {s->batch, s->nk, s->k_heads};
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = qn[i] > 1 ? s->q_stride[i] : 0; a.gs[i] = qn[i] > 1 ? s->g_stride[i] : 0;
        a.ks[i] = kn[i] > 1 ? s->k_stride[i] : 0; a.vs[i] = kn[i] > 1 ? s->v_stride[i] : 0;
    }
    a.batch = (int)s->batch; a.nq = (int)s->nq; a.nk = (int)s->nk; a.hq = (int)s->q_heads; a.hk = (int)s->k_heads; a.d = (int)s->d;
    a.scale = s->scale;
    a.c = (float)((double)s->scale * 1.4426950408889634);
    a.slack = fminf(8.f / a.c, 1e30f);
    return a;
}

// the mask's bits at the front of the workspace; what follows them is returned
template <typename T> static void *at_bits(const dg_attn_shape *s, const at_plan &p, const uint8_t *mask, at_args<T> &a, void *ws, hipStream_t st)
{
    if (!p.bits) return ws;
    const int64_t n = s->masks * s->nq * dg_cdiv(s->nk, 1024);
    hipLaunchKernelGGL(k_attn_bits, dg_grid(n), dim3(AT_THREADS), 0, st, mask, s->mask_stride[0], s->mask_stride[1], (u32 *)ws, (u32)n, (int)s->nq, (int)s->nk,
                       (int)p.words);
    a.bits = (const u32 *)ws;
    a.words = (int)p.words;
    a.bs = s->masks > 1 ? s->nq * p.words : 0;
    return (char *)ws + p.bits;
}

#define AT_LAUNCH(kernel, mode, grid, a)                                                                                        \
    do {                                                                                                                        \
        const dim3 gr_((unsigned)(grid)), bl_(AT_THREADS);                                                                       \
        if ((a).d <= 32) hipLaunchKernelGGL((kernel<T, 32, mode>), gr_, bl_, 0, st, a);                                          \
        else if ((a).d <= 64) hipLaunchKernelGGL((kernel<T, 64, mode>), gr_, bl_, 0, st, a);                                     \
        else hipLaunchKernelGGL((kernel<T, 128, mode>), gr_, bl_, 0, st, a);                                                     \
    } while (0)

template <typename T>
static int at_forward(const dg_attn_shape *s, const void *q, const void *k, const void *v, const int32_t *qc, const int32_t *kc, const uint8_t *mask, void *out,
                      float *lse, void *rest, void *ws, hipStream_t st)
{
    const at_plan p = at_plan_of(s);
    at_args<T> a = at_fill<T>(s, q, k, v, qc, kc);
    ws = at_bits(s, p, mask, a, ws, st);
    a.o = (T *)out; a.lse = lse; a.rest = (T *)rest; a.part = (float *)ws;
    a.tiles = (int)p.qtiles; a.splits = (int)p.qsplits; a.per = (int)p.qper;
    if (a.bits) AT_LAUNCH(k_attn_fwd, true, s->batch * s->k_heads * p.qtiles * p.qsplits, a);
    else AT_LAUNCH(k_attn_fwd, false, s->batch * s->k_heads * p.qtiles * p.qsplits, a);
    if (p.qsplits > AT_JOIN_FEW) hipLaunchKernelGGL((k_attn_join<T, true>), dim3((unsigned)(p.rows * dg_cdiv(s->d, 32))), dim3(AT_THREADS), 0, st, a, p.rows);
    else if (p.qsplits > 1) hipLaunchKernelGGL((k_attn_join<T, false>), dim3((unsigned)dg_cdiv(p.rows, 8)), dim3(AT_THREADS), 0, st, a, p.rows);
    DG_CHECK_LAUNCH("k_attn_fwd");
    return DG_OK;
}

extern "C" int dg_roi_attn_fwd(const dg_attn_shape *s, const void *q, const void *k, const void *v, const int32_t *q_counts, const int32_t *k_counts,
                               const uint8_t *mask, void *out, float *lse, void *rest, void *ws, size_t ws_bytes, dg_stream_t stream)
{
    const int rc = at_check(s, "roi_attn_fwd");
    if (rc != DG_OK) return rc;
    if (s->batch == 0 || s->nq == 0) return DG_OK;
    DG_REQUIRE(q && out && lse && (s->nk == 0 || (k && v && !mask == !s->masks)), "roi_attn_fwd: null pointer");
    DG_REQUIRE(!rest || s->dtype == DG_BF16, "roi_attn_fwd: rest is for DG_BF16 only");
    DG_REQUIRE(at_aligned(q, s->q_stride, s, s->nq, s->q_heads) && at_aligned(k, s->k_stride, s, s->nk, s->k_heads) &&
                   at_aligned(v, s->v_stride, s, s->nk, s->k_heads) && ((((uintptr_t)out) | ((uintptr_t)rest)) & 15) == 0, "roi_attn_fwd: pointers and strides must be multiples of 16 bytes, rows at most 2^22 values apart");
    const size_t need = dg_roi_attn_workspace_bytes(s, 0);
    if (ws_bytes < need || (need && !ws)) { dg_set_error("roi_attn_fwd: workspace %zu < %zu bytes", ws_bytes, need); return DG_ENOMEM; }
    DG_REQUIRE((((uintptr_t)ws) & 15) == 0, "roi_attn_fwd: workspace must be 16-byte aligned");
    return s->dtype == DG_F32 ? at_forward<float>(s, q, k, v, q_counts, k_counts, mask, out, lse, rest, ws, (hipStream_t)stream)
                              : at_forward<__bf16>(s, q, k, v, q_counts, k_counts, mask, out, lse, rest, ws, (hipStream_t)stream);
}

template <typename T>
static int at_backward(const dg_attn_shape *s, const void *g, const void *q, const void *k, const void *v, const void *out, const float *lse, const void *rest, const int32_t *qc,
                       const int32_t *kc, const uint8_t *mask, void *dq, void *dk, void *dv, void *ws, hipStream_t st)
{
    const at_plan p = at_plan_of(s);
    at_args<T> a = at_fill<T>(s, q, k, v, qc, kc);
    ws = at_bits(s, p, mask, a, ws, st);
    constexpr int FINE = sizeof(T) == 2 ? AT_FINE : AT_PLAIN, COUNTED = sizeof(T) == 2 ? AT_COUNTED : AT_PLAIN;
    // 16 x 500 rows and keys x 64: dq 36 -> 39 us, dk, dv 47 -> 51, for errors of dq, dk of 1.0 instead of 1.45 roundings of the result (2.3 at 10
    // keys of which a fifth is seen); 16000 x 128: dq 1575 -> 1980, dk, dv 2235 -> 2545, for 1.0 instead of 1.42.  Both walks in one kernel, by
    // count: 8 x 2000 to 1900 x 64 dq 121 -> 118, dk, dv 150 -> 152 (with delta); 4 x 4000 x 128 289 -> 287, 486 -> 497
    const bool fine = s->nk <= AT_FEW;
    f32x2 *stat = (f32x2 *)ws;
    a.g = (const T *)g; a.rest = (T *)rest; a.stat = stat; a.part = (float *)((char *)ws + p.stats);
    if (s->nq > 0) {
        const int64_t rpb = AT_THREADS * (16 / (int64_t)sizeof(T)) / 128;
        const dim3 grid((unsigned)dg_cdiv(p.rows, rpb));
        if (a.bits) hipLaunchKernelGGL((k_attn_delta<T, true>), grid, dim3(AT_THREADS), 0, st, a, (const T *)out, lse, stat, (u32)p.rows);
        else hipLaunchKernelGGL((k_attn_delta<T, false>), grid, dim3(AT_THREADS), 0, st, a, (const T *)out, lse, stat, (u32)p.rows);
    }
    if (s->nq > 0 && dq) {
        a.o = (T *)dq;
        a.tiles = (int)p.qtiles; a.splits = (int)p.qsplits; a.per = (int)p.qper;
        const int64_t grid = s->batch * s->k_heads * p.qtiles * p.qsplits;
        if (a.bits) AT_LAUNCH(k_attn_dq, AT_MASKED, grid, a);
        else if (fine) AT_LAUNCH(k_attn_dq, FINE, grid, a);
        else if (kc) AT_LAUNCH(k_attn_dq, COUNTED, grid, a);
        else AT_LAUNCH(k_attn_dq, AT_PLAIN, grid, a);
        if (p.qsplits > 1)
            hipLaunchKernelGGL((k_attn_sum<T>), dim3((unsigned)dg_cdiv(p.rows * s->d / 4, AT_THREADS)), dim3(AT_THREADS), 0, st, (const float *)a.part, (T *)dq, (T *)nullptr, qc, p.rows,
                               (int)s->q_heads, (int)s->nq, (int)s->d, (int)p.qsplits);
    }
    if (s->nk > 0 && dk) {
        a.dk = (T *)dk; a.dv = (T *)dv;
        a.tiles = (int)p.ktiles; a.splits = (int)p.ksplits; a.per = (int)p.kper;
        const int64_t grid = s->batch * s->k_heads * p.ktiles * p.ksplits;
        if (a.bits) AT_LAUNCH(k_attn_dkv, AT_MASKED, grid, a);
        else if (fine) AT_LAUNCH(k_attn_dkv, FINE, grid, a);
        else if (kc) AT_LAUNCH(k_attn_dkv, COUNTED, grid, a);
        else AT_LAUNCH(k_attn_dkv, AT_PLAIN, grid, a);
        if (p.ksplits > 1) {
            const int64_t rows = s->batch * s->k_heads * s->nk;
            hipLaunchKernelGGL((k_attn_sum<T>), dim3((unsigned)dg_cdiv(rows * s->d / 4, AT_THREADS), 2), dim3(AT_THREADS), 0, st, (const float *)a.part, (T *)dk, (T *)dv,
                               (const int32_t *)nullptr, rows, (int)s->k_heads, (int)s->nk, (int)s->d, (int)p.ksplits);
        }
    }
    DG_CHECK_LAUNCH("k_attn_dkv");
    return DG_OK;
}

extern "C" int dg_roi_attn_bwd(const dg_attn_shape *s, const void *grad_out, const void *q, const void *k, const void *v, const void *out, const float *lse,
                               const void *rest, const int32_t *q_counts, const int32_t *k_counts, const uint8_t *mask, void *dq, void *dk, void *dv, void *ws, size_t ws_bytes,
                               dg_stream_t stream)
{
    const int rc = at_check(s, "roi_attn_bwd");
    if (rc != DG_OK) return rc;
    if (s->batch == 0 || (s->nq == 0 && s->nk == 0)) return DG_OK;
    DG_REQUIRE((s->nq == 0 || (grad_out && q && out && lse)) && (s->nk == 0 || (k && v)) && !dk == !dv && (s->nk == 0 || s->nq == 0 || !mask == !s->masks), "roi_attn_bwd: null pointer");
    DG_REQUIRE(!rest || s->dtype == DG_BF16, "roi_attn_bwd: rest is for DG_BF16 only");
    DG_REQUIRE(at_aligned(q, s->q_stride, s, s->nq, s->q_heads) && at_aligned(k, s->k_stride, s, s->nk, s->k_heads) &&
                   at_aligned(v, s->v_stride, s, s->nk, s->k_heads) && at_aligned(grad_out, s->g_stride, s, s->nq, s->q_heads) &&
                   ((((uintptr_t)out) | ((uintptr_t)rest) | ((uintptr_t)dq) | ((uintptr_t)dk) | ((uintptr_t)dv)) & 15) == 0, "roi_attn_bwd: pointers and strides must be multiples of 16 bytes, rows at most 2^22 values apart");
    const size_t need = dg_roi_attn_workspace_bytes(s, 1);
    if (ws_bytes < need || (need && !ws)) { dg_set_error("roi_attn_bwd: workspace %zu < %zu bytes", ws_bytes, need); return DG_ENOMEM; }
    DG_REQUIRE((((uintptr_t)ws) & 15) == 0, "roi_attn_bwd: workspace must be 16-byte aligned");
    return s->dtype == DG_F32
               ? at_backward<float>(s, grad_out, q, k, v, out, lse, rest, q_counts, k_counts, mask, dq, dk, dv, ws, (hipStream_t)stream)
               : at_backward<__bf16>(s, grad_out, q, k, v, out, lse, rest, q_counts, k_counts, mask, dq, dk, dv, ws, (hipStream_t)stream);
}
