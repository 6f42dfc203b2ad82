// rope.hip — rotary positions over several axes (frame, row, column of a box centre or map cell) for queries and keys.
//   pair j of a token turns by a = pos[token][axis_j] * f_j:  (u, v) -> (u cos a - v sin a, u sin a + v cos a)
// The map is a rotation, so its gradient is the turn by -a: the same kernel.  Values are read once and written once: bound by
// memory: 4 x 30400 tokens, 20 heads of 128 bf16: 212 us, 5.9 TB/s; 16 x 2000, 16 heads of 80 fp32: 70 us, 4.7 TB/s (a copy of 1 GB: 5.0).
// The sines of a token are formed once, by the first phase of its workgroup, and serve all heads of q and k from LDS.
// Angles are held in turns in 64 bits and reduced to [-1/2, 1/2] before they are rounded to 32: a far position (a frame number
// of 10^5) keeps its angle, where a 32-bit product would be off by a hundredth of a radian.
#include "common.hpp"
#include <hip/hip_bf16.h>

typedef u32 rp_u4 __attribute__((ext_vector_type(4)));

struct rp_args {
    const void *x[2];                             // q, k
    void *y[2];
    const void *pos;
    const double *turns;
    const int32_t *axis;
    int64_t xs[2][3], ps[2];                      // strides in values: batch, token, head; pos: batch, token
    u32 tokens, n, heads[2], d, pairs, tok, units;   // tok: tokens of a workgroup, units: pieces of a head
    int axes;
    float sign;
    bool past;
};

template <typename T, int VEC> struct rp_piece { T v[VEC]; };
// past: results that no cache would hold until they are read (with the inputs more than the 256 MB of the last one) are written around
// it: 16 x 2000, 16 heads of 80 fp32 73.5 -> 70 us, 4 x 30400, 20 heads of 128 bf16 218 -> 212
template <typename P, typename T> __device__ __forceinline__ void rp_put(T *y, const P &o, bool past)
{
    if constexpr (sizeof(P) == 16) {
        if (past) { __builtin_nontemporal_store(__builtin_bit_cast(rp_u4, o), (rp_u4 *)y); return; }
    }
    *(P *)y = o;
}

// a piece: VEC pairs (halves) or VEC values (neighbours) that turn, or VEC values behind the turned ones, copied as they are
template <typename T, typename P, int VEC, bool HALVES>
__global__ __launch_bounds__(256) void k_rope_axes(const rp_args a)
{
    typedef rp_piece<T, VEC> piece;
    extern __shared__ float2 cs[];                // [tok][pairs]
    const u32 t0 = dg_block() * a.tok;            // tokens number fewer than 2^31
    if (t0 >= a.tokens) return;
    const u32 nt = min(a.tok, a.tokens - t0);
    for (u32 i = threadIdx.x; i < nt * a.pairs; i += 256) {
        const u32 t = i / a.pairs, j = i - t * a.pairs, b = (t0 + t) / a.n, n = t0 + t - b * a.n;
        const int ax = min(max(a.axis[j], 0), a.axes - 1);
        double r = (double)((const P *)a.pos)[b * a.ps[0] + n * a.ps[1] + ax] * a.turns[j];
        r -= rint(r);
        float s, c;
        sincospif(2.0f * (float)r, &s, &c);
        cs[i] = make_float2(c, s * a.sign);
    }
    __syncthreads();
    const u32 per = a.units * (a.heads[0] + a.heads[1]), turning = (HALVES ? a.pairs : 2 * a.pairs) / VEC;
    for (u32 i = threadIdx.x; i < nt * per; i += 256) {
        const u32 t = i / per, r = i - t * per, hh = r / a.units, u = r - hh * a.units;
        const u32 w = hh >= a.heads[0], h = w ? hh - a.heads[0] : hh, b = (t0 + t) / a.n, n = t0 + t - b * a.n;
        const T *x = (const T *)a.x[w] + b * a.xs[w][0] + n * a.xs[w][1] + h * a.xs[w][2];
        T *y = (T *)a.y[w] + ((int64_t)(t0 + t) * a.heads[w] + h) * a.d;
        const float2 *c = cs + t * a.pairs;
        if (HALVES) {
            if (u < turning) {
                const u32 j = u * VEC;
                const piece p = *(const piece *)(x + j), q = *(const piece *)(x + a.pairs + j);
                piece o, s;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 k = c[j + e];
                    const float pv = (float)p.v[e], qv = (float)q.v[e];
                    o.v[e] = (T)fmaf(pv, k.x, -(qv * k.y));
                    s.v[e] = (T)fmaf(pv, k.y, qv * k.x);
                }
                rp_put(y + j, o, a.past);
                rp_put(y + a.pairs + j, s, a.past);
            } else {
                const u32 j = 2 * a.pairs + (u - turning) * VEC;
                rp_put(y + j, *(const piece *)(x + j), a.past);
            }
        } else {
            const u32 j = u * VEC;
            piece p = *(const piece *)(x + j);
            if (u < turning) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 k = c[(j + e) >> 1];
                    const float pv = (float)p.v[e], qv = (float)p.v[e + 1];
                    p.v[e] = (T)fmaf(pv, k.x, -(qv * k.y));
                    p.v[e + 1] = (T)fmaf(pv, k.y, qv * k.x);
                }
            }
            rp_put(y + j, p, a.past);
        }
    }
}

// 16 bytes at a time where pointers, strides and the cut points of a head allow it, single values (pairs) elsewhere
template <typename T, typename P>
static void rp_launch(const rp_args &a0, bool halves, hipStream_t st)
{
    rp_args a = a0;
    constexpr int V = 16 / (int)sizeof(T);
    bool wide = a.d % V == 0 && (halves ? a.pairs : 2 * a.pairs) % V == 0;
    for (int w = 0; w < 2; ++w) {
        if (!a.heads[w]) continue;
        wide &= ((((uintptr_t)a.x[w]) | ((uintptr_t)a.y[w])) & 15) == 0;
        for (int i = 0; i < 3; ++i) wide &= a.xs[w][i] % V == 0;
    }
    a.tok = 1;
    while (a.tok < 16 && a.tok * a.pairs < 256) a.tok *= 2;
    const dim3 grid = dg_grid(dg_cdiv(a.tokens, a.tok)), block(256);
    const size_t lds = (size_t)a.tok * a.pairs * sizeof(float2);
    const u32 rest = a.d - 2 * a.pairs;
    if (halves) {
        a.units = wide ? (a.pairs + rest) / V : a.pairs + rest;
        if (wide) hipLaunchKernelGGL((k_rope_axes<T, P, V, true>), grid, block, lds, st, a);
        else hipLaunchKernelGGL((k_rope_axes<T, P, 1, true>), grid, block, lds, st, a);
    } else {
        a.units = wide ? a.d / V : a.d / 2;
        if (wide) hipLaunchKernelGGL((k_rope_axes<T, P, V, false>), grid, block, lds, st, a);
        else hipLaunchKernelGGL((k_rope_axes<T, P, 2, false>), grid, block, lds, st, a);
    }
}

extern "C" int dg_rope_axes(const dg_rope_shape *s, const void *q, const void *k, const void *pos, const double *turns, const int32_t *axis, int inverse,
                            void *out_q, void *out_k, dg_stream_t stream)
{
    DG_REQUIRE(s, "rope_axes: null shape");
    DG_REQUIRE(s->dtype == DG_F32 || s->dtype == DG_BF16 || s->dtype == DG_F16, "rope_axes: type must be DG_F32, DG_BF16 or DG_F16");
    DG_REQUIRE(s->pos_dtype == DG_F32 || s->pos_dtype == DG_F64, "rope_axes: positions must be DG_F32 or DG_F64");
    const int64_t most = 1ll << 20;
    DG_REQUIRE(s->batch >= 0 && s->n >= 0 && s->n < (1ll << 31) && s->batch < (1ll << 31), "rope_axes: bad batch or token count");
    DG_REQUIRE(s->q_heads >= 0 && s->k_heads >= 0 && s->q_heads + s->k_heads >= 1 && s->q_heads <= most && s->k_heads <= most, "rope_axes: bad head count");
    DG_REQUIRE(s->d >= 2 && s->d <= 4096 && s->d % 2 == 0, "rope_axes: head size %lld is not even or not from 2 to 4096", (long long)s->d);
    DG_REQUIRE(s->pairs >= 1 && 2 * s->pairs <= s->d, "rope_axes: %lld pairs do not fit a head of %lld", (long long)s->pairs, (long long)s->d);
    DG_REQUIRE(s->axes >= 1 && s->axes <= 16, "rope_axes: 1 to 16 axes");
    DG_REQUIRE(s->pairing == DG_ROPE_HALVES || s->pairing == DG_ROPE_NEIGHBOURS, "rope_axes: unknown pairing");
    const int64_t tokens = s->batch * s->n;
    DG_REQUIRE(tokens < (1ll << 31) && (s->q_heads + s->k_heads) * s->d * 16 < (1ll << 31), "rope_axes: too large");
    if (tokens == 0) return DG_OK;
    DG_REQUIRE(pos && turns && axis && (!s->q_heads || (q && out_q)) && (!s->k_heads || (k && out_k)), "rope_axes: null pointer");
    rp_args a = {};
    a.x[0] = q; a.x[1] = k; a.y[0] = out_q; a.y[1] = out_k;
    a.pos = pos; a.turns = turns; a.axis = axis;
    for (int i = 0; i < 3; ++i) { a.xs[0][i] = s->q_stride[i]; a.xs[1][i] = s->k_stride[i]; }
    a.ps[0] = s->pos_stride[0]; a.ps[1] = s->pos_stride[1];
    a.tokens = (u32)tokens; a.n = (u32)s->n; a.heads[0] = (u32)s->q_heads; a.heads[1] = (u32)s->k_heads;
    a.past = tokens * (s->q_heads + s->k_heads) * s->d * (s->dtype == DG_F32 ? 4 : 2) > (1ll << 27);
    a.d = (u32)s->d; a.pairs = (u32)s->pairs; a.axes = (int)s->axes; a.sign = inverse ? -1.f : 1.f;
    const bool halves = s->pairing == DG_ROPE_HALVES, p64 = s->pos_dtype == DG_F64;
    hipStream_t st = (hipStream_t)stream;
    if (s->dtype == DG_F32) p64 ? rp_launch<float, double>(a, halves, st) : rp_launch<float, float>(a, halves, st);
    else if (s->dtype == DG_BF16) p64 ? rp_launch<__bf16, double>(a, halves, st) : rp_launch<__bf16, float>(a, halves, st);
    else p64 ? rp_launch<_Float16, double>(a, halves, st) : rp_launch<_Float16, float>(a, halves, st);
    DG_CHECK_LAUNCH("k_rope_axes");
    return DG_OK;
}
