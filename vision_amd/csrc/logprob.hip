// logprob.hip — log probabilities of given classes, with entropy and the best alternatives, and their gradient.
//   l = log sum_j e^z_j,  logp = z_y - l,  H = log s - w / s  with  s = sum e^(z-m), w = sum e^(z-m) (z-m), m = max z
//   dz_j = g (1[j = y] - p_j) - gH p_j (z_j - l + H),  p_j = e^(z_j - l)
// The entropy is formed from differences to the maximum (not from l - sum p z), so that large scores of one row cost no digits.
// For the same reason l is kept as the pair (m, log s), and log probabilities are (z - m) - log s.
// The forward pass reads the scores once: maximum, sums and the list of the best run along together.  Bound by memory.
#include "common.hpp"
#include <hip/hip_bf16.h>
#include <math.h>

#define LP_LOG2E 1.4426950408889634f
#define LP_NONE (~0ull)

struct lp_args {
    const void *z;
    const int64_t *y;                             // may be NULL
    int64_t n, c, stride;                         // stride of a row in values
    float *logp, *entropy, *norm, *top_logp;      // logp and entropy may be NULL; norm: pairs
    int64_t *top_index;
    int32_t *status;
    u64 *keys;                                    // partial results of split rows
    float *part;
    int64_t per;                                  // classes of a split
    int top, splits;
};

// order of the best: larger scores first (-0 and 0 are one value), equal ones by index, NaN behind -inf
__device__ __forceinline__ u32 lp_desc(float v) { return v != v ? 0xfffffffeu : dg_score_desc(v + 0.0f); }
__device__ __forceinline__ u64 lp_key(float v, u32 j) { return ((u64)lp_desc(v) << 32) | j; }
__device__ __forceinline__ float lp_value(u64 key)
{
    const u32 ord = ~(u32)(key >> 32);
    return __uint_as_float((ord & 0x80000000u) ? ord & 0x7fffffffu : ~ord);
}
__device__ __forceinline__ u64 lp_lane(u64 v, int l)
{
    return ((u64)(u32)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) | (u32)__builtin_amdgcn_readlane((int)v, l);
}

// maximum over the wave, by lane moves of the vector unit: 1, 2, 4, 8 lanes on inside sixteen, then across; the last lane has it
template <int MOVE> __device__ __forceinline__ float lp_max_move(float v)
{
    return fmaxf(v, __uint_as_float((u32)__builtin_amdgcn_update_dpp((int)0xff800000, (int)__float_as_uint(v), MOVE, 0xf, 0xf, false)));
}
__device__ __forceinline__ float lp_wave_max(float v)
{
    v = lp_max_move<0x111>(v);                    // row_shr:1, 2, 4, 8
    v = lp_max_move<0x112>(v);
    v = lp_max_move<0x114>(v);
    v = lp_max_move<0x118>(v);
    v = lp_max_move<0x142>(v);                    // row_bcast:15, 31
    v = lp_max_move<0x143>(v);
    return __uint_as_float((u32)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// every lane's value to the lane behind it (the first lane's result is no one's)
__device__ __forceinline__ u64 lp_behind(u64 v)
{
    const u32 lo = (u32)__builtin_amdgcn_update_dpp(0, (int)(u32)v, 0x138, 0xf, 0xf, false), hi = (u32)__builtin_amdgcn_update_dpp(0, (int)(u32)(v >> 32), 0x138, 0xf, 0xf, false);
    return ((u64)hi << 32) | lo;                  // wave_shr:1
}

// the best keys seen by a wave, ascending (best first): lane i holds the i-th
struct lp_list {
    u64 list = LP_NONE, thr = LP_NONE;
    __device__ __forceinline__ void offer(u64 key, int keep, int lane)
    {
        u64 some = __ballot(key < thr);
        while (some) {
            const int l = __ffsll((unsigned long long)some) - 1;
            const u64 c = lp_lane(key, l), up = lp_behind(list);
            list = list < c ? list : (lane == 0 || up < c) ? c : up;
            thr = lp_lane(list, keep - 1);
            if (lane == l) key = LP_NONE;
            some = __ballot(key < thr);
        }
    }
};

// statistics of a set of scores: maximum, sum of e^(z-m), sum of e^(z-m) (z-m); far: the part of the sums that has been put away.  The
// roundings of a sum of thousands of like terms all point one way (131072 classes in one sum a lane: 2e-5 of a log probability was
// lost), so a walk adds a turn's terms up first and puts sixteen turns away together.
struct lp_sum {
    float m = -INFINITY, s = 0.f, w = 0.f, far_s = 0.f, far_w = 0.f;
    __device__ __forceinline__ void raise(float mx)
    {
        if (mx > m) {
            const float d = m - mx, f = __builtin_amdgcn_exp2f(d * LP_LOG2E);
            w = f == 0.f ? 0.f : f * fmaf(s, d, w);
            s *= f;
            far_w = f == 0.f ? 0.f : f * fmaf(far_s, d, far_w);
            far_s *= f;
            m = mx;
        }
    }
    __device__ __forceinline__ void put_away()
    {
        far_s += s;
        far_w += w;
        s = w = 0.f;
    }
    __device__ __forceinline__ void take_back()
    {
        s += far_s;
        w += far_w;
        far_s = far_w = 0.f;
    }
    __device__ __forceinline__ float from() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void add(float z, float from)  // z <= m, or NaN
    {
        const float d = z - from, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        s += e;
        w = fmaf(e, fmaxf(d, -3.0e38f), w);
    }
    __device__ __forceinline__ void join(float om, float os, float ow)
    {
        const float mx = fmaxf(m, om);
        if (mx == -INFINITY) { s += os; return; } // nothing on either side, or only NaN
        const float a = m - mx, b = om - mx;
        const float fa = __builtin_amdgcn_exp2f(a * LP_LOG2E), fb = __builtin_amdgcn_exp2f(b * LP_LOG2E);
        const float wa = fa == 0.f ? 0.f : fa * fmaf(s, a, w), wb = fb == 0.f ? 0.f : fb * fmaf(os, b, ow);
        s = fa * s + fb * os;
        w = wa + wb;
        m = mx;
    }
    template <int L> __device__ __forceinline__ void join_lanes()
    {
#pragma unroll
        for (int x = L / 2; x; x >>= 1) {
            const float om = __shfl_xor(m, x, 64), os = __shfl_xor(s, x, 64), ow = __shfl_xor(w, x, 64);
            join(om, os, ow);
        }
    }
    __device__ __forceinline__ float entropy() const { return s == 0.f ? 0.f : fmaxf(logf(s) - w / s, 0.f) + (s - s); }
};

// what turns a score into a log probability; a row with nothing to choose from (all -inf): -inf throughout, entropy 0
struct lp_norm {
    float m, ls;
    __device__ __forceinline__ explicit lp_norm(const lp_sum &t) : m(t.m), ls(t.s == 0.f ? 0.f : logf(t.s)) {}
    __device__ __forceinline__ lp_norm(float m_, float ls_) : m(m_), ls(ls_) {}
    __device__ __forceinline__ float of(float z) const { return m == -INFINITY && ls == 0.f ? -INFINITY : (z - m) - ls; }
};

// the numbers of a row beside its best: one lane writes them
template <typename T>
__device__ __forceinline__ void lp_write(const lp_args &a, int64_t row, const lp_sum &t, const lp_norm &nm)
{
    if (a.entropy) a.entropy[row] = t.entropy();
    a.norm[2 * row] = nm.m;
    a.norm[2 * row + 1] = nm.ls;
    if (a.y) {
        const int64_t y = a.y[row];
        float v = 0.f;                            // a negative label: no class given
        if (y >= a.c) { v = __builtin_nanf(""); if (a.status) atomicOr(a.status, 1); }
        else if (y >= 0) v = nm.of((float)((const T *)a.z)[row * a.stride + y]);
        a.logp[row] = v;
    }
}

// ------------------------------------------------------------------ up to 512 classes: L lanes hold a row, 8 scores each
// (32000 x 81 fp32, the best 3: 10 us; the rows of a wave and the rounds over its best bound it, not the 10 MB)
template <typename T, int L>
__global__ __launch_bounds__(256) void k_logprob_small(const lp_args a)
{
    const int sub = threadIdx.x & (L - 1);
    const int64_t row = (int64_t)dg_block() * (256 / L) + threadIdx.x / L;
    if (row >= a.n) return;                       // whole groups: shuffles stay among the lanes of a row
    const T *z = (const T *)a.z + row * a.stride;
    float v[8];
    lp_sum t;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int j = sub + i * L;
        v[i] = j < a.c ? (float)z[j] : -INFINITY;
        mx = fmaxf(mx, v[i]);
    }
#pragma unroll
    for (int x = L / 2; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
    t.raise(mx);
#pragma unroll
    for (int i = 0; i < 8; ++i) t.add(v[i], t.from());
#pragma unroll
    for (int x = L / 2; x; x >>= 1) {             // one maximum for all lanes: the sums just add up
        t.s += __shfl_xor(t.s, x, 64);
        t.w += __shfl_xor(t.w, x, 64);
    }
    const lp_norm nm(t);
    if (sub == 0) lp_write<T>(a, row, t, nm);
    if (a.top == 0) return;
    u32 key[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) key[i] = sub + i * L < a.c ? lp_desc(v[i]) : 0xffffffffu;
    for (int r = 0; r < a.top; ++r) {
        u32 best = 0xffffffffu, at = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (key[i] < best) { best = key[i]; at = i; }
        u32 j = sub + at * L;
#pragma unroll
        for (int x = L / 2; x; x >>= 1) {
            const u32 ob = __shfl_xor(best, x, 64), oj = __shfl_xor(j, x, 64);
            if (ob < best || (ob == best && oj < j)) { best = ob; j = oj; }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j == (u32)(sub + i * L)) key[i] = 0xffffffffu;
        if (sub == 0) {
            a.top_logp[row * a.top + r] = nm.of(lp_value((u64)best << 32));
            a.top_index[row * a.top + r] = j;
        }
    }
}

// ------------------------------------------------------------------ more classes: waves walk a row
__device__ __forceinline__ void lp_best(const lp_args &a, int64_t row, const lp_list &b, const lp_norm &n, int lane)
{
    if (lane < a.top) {
        a.top_logp[row * a.top + lane] = n.of(lp_value(b.list));
        a.top_index[row * a.top + lane] = (u32)b.list;
    }
}

// 8192 x 20011 bf16: 87 us, 3.8 TB/s (maximum, three sums and the comparisons, about ten operations a score, bound it); 4096 x 32000
// fp32: 99 us, 5.3 TB/s, the rate of a copy.  Sixteen scores a lane and turn: with 32 of them fewer waves fit (100 us).
// WPR waves walk one row's split (4: a workgroup, 1: each wave a row of its own).  Scores come 16 bytes at a time from the first
// aligned one on; the few before and behind are single loads.
template <typename T, int WPR>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? 8 : 6)) void k_logprob_walk(const lp_args a)
{
    constexpr int V = 16 / (int)sizeof(T), UN = 16 / V;
    typedef T vec __attribute__((ext_vector_type(V)));
    __shared__ float sums[4][3];
    __shared__ u64 lists[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = WPR == 4 ? threadIdx.x : lane;
    const int64_t part = WPR == 4 ? dg_block() : (int64_t)dg_block() * 4 + wave;
    const int64_t row = part / a.splits, sp = part - row * a.splits;
    if (row >= a.n) return;                       // WPR == 1: whole waves, and no barrier follows
    const int keep = a.top;
    const T *z = (const T *)a.z + row * a.stride;
    const int64_t c0 = sp * a.per, c1 = min(a.c, c0 + a.per);
    // first aligned class of the split, last whole piece
    int64_t b0 = c0 + (int64_t)(((16 - ((uintptr_t)(z + c0) & 15)) & 15) / sizeof(T));
    if (b0 > c1) b0 = c1;
    const int64_t pieces = (c1 - b0) / V, b1 = b0 + pieces * V;

    lp_sum t;
    lp_list best;
    auto single = [&](int64_t from, int64_t to) { // what lies before the first piece or behind the last: under V scores each
        const int64_t j = from + lane;
        const float v = j < to ? (float)z[j] : -INFINITY;
        t.raise(v);
        if (j < to) t.add(v, t.from());
        if (keep) best.offer(j < to ? lp_key(v, (u32)j) : LP_NONE, keep, lane);
    };
    if (wave == 0 || WPR == 1) single(c0, b0);
    const vec *zp = (const vec *)(z + b0);
    vec next[UN];                                 // the following turn's pieces are on their way while this one's are summed
    auto fetch = [&](int64_t p0) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int64_t p = p0 + u * (64 * WPR) + tid;
            if (p < pieces) next[u] = zp[p];
        }
    };
    fetch(0);
    for (int64_t p0 = 0; p0 < pieces; p0 += 64 * WPR * UN) {
        float v[UN][V];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int64_t p = p0 + u * (64 * WPR) + tid;
            if (p < pieces) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[u][e] = (float)next[u][e];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) v[u][e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) mx = fmaxf(mx, v[u][e]);
        }
        fetch(p0 + 64 * WPR * UN);
        t.raise(mx);
        const float from = t.from();
        lp_sum turn;
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) turn.add(v[u][e], from);
        t.s += turn.s;
        t.w += turn.w;
        if ((p0 & (64 * WPR * UN * 15)) == 64 * WPR * UN * 15) t.put_away();
        if (!keep) continue;
        // A score enters the list only from `least` on: the keep-th best so far, or, before there is a list, the keep-th largest of
        // the lanes' maxima -- which leaves little more than the best themselves to be sorted in, not the first ones met.
        float least = lp_value(best.thr);
        if (best.thr == LP_NONE) {
            float x = mx;
            for (int i = 0; i < keep; ++i) {
                least = lp_wave_max(x);
                if (lane == __ffsll((unsigned long long)__ballot(x == least)) - 1) x = -INFINITY;
            }
        } else if (!__any(!(mx <= least))) continue; // later classes rank behind equal ones (before a list of NaN all do)
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int64_t p = p0 + u * (64 * WPR) + tid;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (__any(!(v[u][e] < least))) best.offer(p < pieces ? lp_key(v[u][e], (u32)(b0 + p * V + e)) : LP_NONE, keep, lane);
        }
    }
    if (wave == 0 || WPR == 1) single(b1, c1);    // in the order of the classes: an equal score that comes later never ranks before
    t.take_back();
    t.join_lanes<64>();
    if (WPR == 4) {
        if (lane == 0) { sums[wave][0] = t.m; sums[wave][1] = t.s; sums[wave][2] = t.w; }
        if (keep) lists[wave][lane] = best.list;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            t.join(sums[i][0], sums[i][1], sums[i][2]);
            if (keep) best.offer(lane < keep ? lists[i][lane] : LP_NONE, keep, lane);
        }
    }
    if (a.splits > 1) {
        if (lane == 0) {
            float *o = a.part + part * 3;
            o[0] = t.m; o[1] = t.s; o[2] = t.w;
        }
        if (lane < keep) a.keys[part * keep + lane] = best.list;
        return;
    }
    const lp_norm nm(t);
    if (lane == 0) lp_write<T>(a, row, t, nm);
    if (a.top) lp_best(a, row, best, nm, lane);
}

// joins the splits of a row: one wave per row
template <typename T>
__global__ __launch_bounds__(64) void k_logprob_join(const lp_args a)
{
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int keep = a.top;
    lp_sum t;
    for (int s = lane; s < a.splits; s += 64) {
        const float *p = a.part + (row * a.splits + s) * 3;
        t.join(p[0], p[1], p[2]);
    }
    t.join_lanes<64>();
    const lp_norm nm(t);
    if (lane == 0) lp_write<T>(a, row, t, nm);
    if (!keep) return;
    lp_list best;
    const u64 *k = a.keys + row * a.splits * keep;
    for (int i0 = 0; i0 < a.splits * keep; i0 += 64) best.offer(i0 + lane < a.splits * keep ? k[i0 + lane] : LP_NONE, keep, lane);
    lp_best(a, row, best, nm, lane);
}

// ------------------------------------------------------------------ backward: one read, one write
// VEC values of the dense gradient, in one list over all rows so that odd numbers of classes stay aligned; a thread that crosses
// the end of a row takes up the next one's numbers.  UN pieces of a thread, 256 apart: four where there is enough for all CUs (8192 x
// 20011 bf16: 143 us, 4.6 TB/s, the rate of a copy; 164 with one), one for small calls (32000 x 81 fp32: 9 us; 12 with four).
template <typename T, int VEC, bool DENSE, int UN>
__global__ __launch_bounds__(256) void k_logprob_bwd(const T *__restrict__ z, const int64_t *__restrict__ y, int64_t n, int64_t c, int64_t stride,
                                                     const float *__restrict__ norm, const float *__restrict__ entropy, const float *__restrict__ g,
                                                     const float *__restrict__ gh, T *__restrict__ dz)
{
    typedef T vec __attribute__((ext_vector_type(VEC)));
    const int64_t end = n * c, first = ((int64_t)dg_block() * (256 * UN) + threadIdx.x) * VEC;
    vec x[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int64_t i0 = first + u * (256 * VEC);
        if (DENSE && i0 + VEC <= end) x[u] = *(const vec *)(z + i0);
    }
    int64_t row = -1, lab = -1;
    lp_norm nm(0.f, 0.f);
    float h = 0.f, gH = 0.f, gl = 0.f;
    auto take = [&](int64_t r) {
        row = r;
        nm = lp_norm(norm[2 * row], norm[2 * row + 1]);
        h = gh ? entropy[row] : 0.f;
        gH = gh ? gh[row] : 0.f;
        lab = y ? y[row] : -1;
        gl = g && lab >= 0 ? g[row] : 0.f;
        if (lab >= c) gl = __builtin_nanf("");
    };
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int64_t i0 = first + u * (256 * VEC);
        if (i0 >= end) return;
        const int64_t r = end < (1ll << 32) ? (int64_t)((u32)i0 / (u32)c) : i0 / c;
        if (r != row) take(r);
        int64_t j = i0 - row * c;
        const bool whole = i0 + VEC <= end;
        vec o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (i0 + e >= end) break;
            const float lp = nm.of(DENSE && whole ? (float)x[u][e] : (float)z[row * stride + j]), p = __builtin_amdgcn_exp2f(lp * LP_LOG2E);
            float v = p == 0.f ? 0.f : -p * fmaf(gH, lp + h, gl);
            if (lab >= c) v = gl;
            if (j == lab && nm.m != -INFINITY) v += gl;
            o[e] = (T)v;
            if (!whole) dz[i0 + e] = o[e];
            if (++j == c && e + 1 < VEC && row + 1 < n) {
                j = 0;
                take(row + 1);
            }
        }
        if (whole) *(vec *)(dz + i0) = o;
    }
}

// ------------------------------------------------------------------ host
static int lp_check(int64_t n, int64_t c, int64_t stride, int dtype, int64_t top, const char *who)
{
    DG_REQUIRE(dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16, "%s: type must be DG_F32, DG_BF16 or DG_F16", who);
    DG_REQUIRE(n >= 0 && n < (1ll << 31), "%s: bad row count", who);
    DG_REQUIRE(c >= 1 && c < (1ll << 31), "%s: 1 to 2^31 - 1 classes", who);
    DG_REQUIRE(stride >= 0, "%s: negative stride", who);
    DG_REQUIRE(top >= 0 && top <= 32 && top <= c, "%s: 0 to 32 alternatives, no more than classes", who);
    return DG_OK;
}

// rows that are too few to fill the chip are split over their classes, 512 workgroups' worth but one split for 4096 classes at most: 2112
// classes or more each (a multiple of 64), the last one what is left, a single class at the least
static void lp_split(int64_t n, int64_t c, int64_t *splits, int64_t *per)
{
    int64_t s = n > 0 && n < 256 ? dg_cdiv(512, n) : 1;
    if (s > dg_cdiv(c, 4096)) s = dg_cdiv(c, 4096);
    *per = dg_round_up(dg_cdiv(c, s), 64);
    *splits = dg_cdiv(c, *per);
}

extern "C" size_t dg_class_logprobs_workspace_bytes(int64_t n, int64_t c, int64_t top)
{
    if (n <= 0 || c <= 512 || top < 0 || top > 32) return 0;
    int64_t s, per;
    lp_split(n, c, &s, &per);
    return s > 1 ? (size_t)(n * s * (top * 8 + 12)) : 0;
}

template <typename T> static void lp_forward(lp_args &a, hipStream_t st)
{
    if (a.c <= 512) {
#define LP_SMALL(L) hipLaunchKernelGGL((k_logprob_small<T, L>), dg_grid(dg_cdiv(a.n, 256 / L)), dim3(256), 0, st, a)
        if (a.c <= 32) LP_SMALL(4);
        else if (a.c <= 64) LP_SMALL(8);
        else if (a.c <= 128) LP_SMALL(16);
        else if (a.c <= 256) LP_SMALL(32);
        else LP_SMALL(64);
        return;
    }
    // a wave a row where rows alone give every SIMD four waves, or where a row is short; four waves a row elsewhere
    if (a.splits == 1 && (a.c <= 4096 || a.n >= 4096)) hipLaunchKernelGGL((k_logprob_walk<T, 1>), dg_grid(dg_cdiv(a.n, 4)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_logprob_walk<T, 4>), dim3((unsigned)(a.n * a.splits)), dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL((k_logprob_join<T>), dim3((unsigned)a.n), dim3(64), 0, st, a);
}

extern "C" int dg_class_logprobs(const void *logits, int dtype, const int64_t *labels, int64_t n, int64_t c, int64_t stride, int64_t top, float *logp,
                                 float *entropy, float *norm, float *top_logp, int64_t *top_index, int32_t *status, void *ws, size_t ws_bytes, dg_stream_t s)
{
    const int rc = lp_check(n, c, stride, dtype, top, "class_logprobs");
    if (rc != DG_OK) return rc;
    if (n == 0) return DG_OK;
    DG_REQUIRE(logits && norm && (!labels || logp) && (!top || (top_logp && top_index)), "class_logprobs: null pointer");
    DG_REQUIRE((((uintptr_t)logits) & (dtype == DG_F32 ? 3 : 1)) == 0, "class_logprobs: logits are not aligned to their type");
    const size_t need = dg_class_logprobs_workspace_bytes(n, c, top);
    if (ws_bytes < need || (need && !ws)) { dg_set_error("class_logprobs: workspace %zu < %zu bytes", ws_bytes, need); return DG_ENOMEM; }
    DG_REQUIRE((((uintptr_t)ws) & 7) == 0, "class_logprobs: workspace must be 8-byte aligned");
    lp_args a = {};
    a.z = logits; a.y = labels; a.n = n; a.c = c; a.stride = stride;
    a.logp = logp; a.entropy = entropy; a.norm = norm; a.top_logp = top_logp; a.top_index = top_index; a.status = status;
    a.top = (int)top;
    int64_t sp = 1, per = c;
    if (c > 512) lp_split(n, c, &sp, &per);
    a.splits = (int)sp; a.per = per;
    a.keys = (u64 *)ws;
    a.part = (float *)((char *)ws + (size_t)(n * sp * top * 8));
    if (dtype == DG_F32) lp_forward<float>(a, (hipStream_t)s);
    else if (dtype == DG_BF16) lp_forward<__bf16>(a, (hipStream_t)s);
    else lp_forward<_Float16>(a, (hipStream_t)s);
    DG_CHECK_LAUNCH("k_logprob");
    return DG_OK;
}

template <typename T>
static int lp_backward(const void *z, const int64_t *y, int64_t n, int64_t c, int64_t stride, const float *norm, const float *entropy, const float *g, const float *gh,
                       void *dz, hipStream_t st)
{
    constexpr int V = 16 / (int)sizeof(T);
    const bool wide = (((uintptr_t)dz) & 15) == 0, dense = stride == c && (((uintptr_t)z) & 15) == 0;
    const bool many = wide && n * c >= (1ll << 24);
    const int64_t blocks = dg_cdiv(n * c, 256 * (many ? 4 * V : wide ? V : 1));
    DG_REQUIRE(blocks < (1ll << 31), "class_logprobs_bwd: too large");
#define LP_BWD(VEC, DENSE, UN) hipLaunchKernelGGL((k_logprob_bwd<T, VEC, DENSE, UN>), dg_grid(blocks), dim3(256), 0, st, (const T *)z, y, n, c, stride, norm, entropy, g, gh, (T *)dz)
    if (many && dense) LP_BWD(V, true, 4);
    else if (many) LP_BWD(V, false, 4);
    else if (wide && dense) LP_BWD(V, true, 1);
    else if (wide) LP_BWD(V, false, 1);
    else LP_BWD(1, false, 1);
    DG_CHECK_LAUNCH("k_logprob_bwd");
    return DG_OK;
}

extern "C" int dg_class_logprobs_bwd(const void *logits, int dtype, const int64_t *labels, int64_t n, int64_t c, int64_t stride, const float *norm, const float *entropy,
                                     const float *grad_logp, const float *grad_entropy, void *grad_logits, dg_stream_t s)
{
    const int rc = lp_check(n, c, stride, dtype, 0, "class_logprobs_bwd");
    if (rc != DG_OK) return rc;
    if (n == 0) return DG_OK;
    DG_REQUIRE(logits && norm && grad_logits && (!grad_logp || labels) && (!grad_entropy || entropy), "class_logprobs_bwd: null pointer");
    DG_REQUIRE(((((uintptr_t)logits) | ((uintptr_t)grad_logits)) & (dtype == DG_F32 ? 3 : 1)) == 0, "class_logprobs_bwd: not aligned to the type");
    hipStream_t st = (hipStream_t)s;
    if (dtype == DG_F32) return lp_backward<float>(logits, labels, n, c, stride, norm, entropy, grad_logp, grad_entropy, grad_logits, st);
    if (dtype == DG_BF16) return lp_backward<__bf16>(logits, labels, n, c, stride, norm, entropy, grad_logp, grad_entropy, grad_logits, st);
    return lp_backward<_Float16>(logits, labels, n, c, stride, norm, entropy, grad_logp, grad_entropy, grad_logits, st);
}
