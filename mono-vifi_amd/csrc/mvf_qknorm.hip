// mvf_qknorm.hip -- the norm of every query and key head with the position rotation in the same pass, forward and backward.
//
//     n = x * rsqrt(mean(x^2) + eps) * w          per (sequence, token, head), over its D channels
//     y = R(pos) n                                 pairs (a, b) of the first `rot` channels: (a cos t - b sin t, a sin t + b cos t)
//
// The rotated channels are `axes` equal blocks of ra = rot / axes channels, one per coordinate of the position (an index; row
// and column; frame, row and column); pair j of a block turns by t = pos * base^(-2j/ra).  Pairs are neighbours (2j, 2j + 1) or
// halves (j, j + ra/2) of the block.  Backward, with u = R(-pos) dy and r = rsqrt(mean(x^2) + eps):
//     dw = sum over rows of u x r,    dx = r w u - x r^3 / D * sum(u w x)
//
// A frequency is a 64-bit fixed-point fraction of a turn, so pos * freq modulo one turn is one integer product without an error of its
// own; its top bits give the quadrant and a remainder of at most an eighth of a turn, to which the Taylor polynomials of sine
// (x^9) and cosine (x^10) apply with an error below an fp32 step.  What is left is the frequency's rounding, |pos| * 2^-64 of a turn at
// most (base >= 1): below an fp32 step up to |pos| = 2^37, 4e-7 radians at 2^40, 1e-4 at 2^48.  (A product in fp32 loses the angle
// altogether at far positions: half a step of 300,000 is a sixtieth of a radian.)
//
// Bound by memory: 2 passes over the rows forward, 3 backward (12 x (7,680 + 15,360) tokens of 8 x 64 bf16, two axes: 111 us = 5.1 TB/s
// and 199 us = 4.3).  Blocks of an odd number of pairs are loaded one channel at a time (three axes of 64 channels: two): 12 x (1,920 +
// 3,840) tokens of 8 x 32 fp32, three axes: 27 us a call = 5.3 TB/s, of 8 x 16: 16 us = 4.4.  A group of lanes owns a token, so the sines and cosines are
// formed once for all its heads; a lane owns the same pairs of every head, loads them in runs of four, two or one, and the sum
// of squares is a butterfly over the group (DPP), for all heads in flight at once.  All arithmetic is fp32; bf16 is rounded once, at the store.
#include "mvf_common.hpp"

using namespace mvf;

namespace {

constexpr int NT = 256;
constexpr int HB = 4, HG = 2;     // heads in flight per lane, forward and backward (two tensors)

// runs of N channels, as aligned as their elements are
template <typename T, int N>
struct Run {
    typedef T V __attribute__((ext_vector_type(N)));
    typedef V U __attribute__((aligned(sizeof(T))));
};

struct Side {
    const void *x, *gy;
    void *y;                      // forward: y; backward: dx ([B, L, H, D] contiguous)
    const float *w;
    const void *pos;
    int64_t s[3], ps;             // strides of x (batch, token, head); positions per sequence (0: shared)
    int L, H, hg, chunks;         // heads of a group, groups of a token
    int64_t groups;               // B * L * chunks
    int64_t blocks;               // workgroups of this side (backward: as many rows of partial weight gradients)
    float *part;
};
struct NormArgs {
    Side side[2];
    uint64_t freq[MVF_ATTN_MAX_D / 2];      // fractions of a turn per unit of position, 2^64 = one turn
    int D, axes, rot, ra;
    int units, rotu;              // units (of PV pairs) of a row; the rotated ones
    int lpr;                      // lanes of a row: power of two >= units
    int pos64, ragged;
    float eps, invD;
};

// sine and cosine of `turn` / 2^64 of a full turn
MVF_DEV void sincos_turn(uint64_t turn, float &s, float &c)
{
    const uint32_t t = (uint32_t)(turn >> 32);
    const uint32_t q = (t + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(t - (q << 30)) * 1.4629180792671596e-09f;         // 2 pi / 2^32: |x| <= pi / 4
    const float z = x * x;
    float p = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    p = fmaf(z, p, 8.3333333e-3f);
    p = fmaf(z, p, -1.6666667e-1f);
    const float sn = fmaf(x * z, p, x);
    float k = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    k = fmaf(z, k, -1.3888889e-3f);
    k = fmaf(z, k, 4.1666667e-2f);
    k = fmaf(z, k, -0.5f);
    const float cs = fmaf(z, k, 1.0f);
    const float a = q & 1 ? cs : sn, b = q & 1 ? sn : cs;
    s = q & 2 ? -a : a;
    c = (q + 1) & 2 ? -b : b;
}

// a lane's share of a row: PV pairs (v[i], v[PV + i]).  NB: pairs are neighbours, the unit is one run of 2 PV channels from c0;
// otherwise two runs of PV from c0 and c1 (channels that are not rotated have no partner: any pairing of them will do)
template <int PV, bool NB>
struct Unit {
    int c0, c1;                   // first channels of the two runs (NB: c1 = c0 + PV); 0 where there is none
    bool live, live1, rot;        // whether the lane has a unit, and that a second run
    float sn[PV], cs[PV];
    MVF_DEV int channel(int i) const { return NB ? c0 + (i < PV ? 2 * i : 2 * (i - PV) + 1) : (i < PV ? c0 + i : c1 + i - PV); }
    MVF_DEV bool has(int i) const { return NB ? (channel(i) - c0 < PV ? live : live1) : (i < PV ? live : live1); }
};

template <int PV, bool NB>
MVF_DEV Unit<PV, NB> unit_of(const NormArgs &a, int u)
{
    Unit<PV, NB> t;
    t.live = u < a.units;
    t.rot = u < a.rotu;
    if (t.rot) {
        const int j = u * PV, per = a.ra / 2, ax = j / per, jj = j - ax * per;
        t.c0 = ax * a.ra + (NB ? 2 * jj : jj);
        t.c1 = NB ? t.c0 + PV : t.c0 + per;
    } else {
        t.c0 = a.rot + (u - a.rotu) * 2 * PV;
        t.c1 = t.c0 + PV;
    }
    t.live1 = t.live && t.c1 < a.D;
    if (!t.live) t.c0 = 0;
    if (!t.live1) t.c1 = 0;
#pragma unroll
    for (int i = 0; i < PV; ++i) { t.sn[i] = 0.0f; t.cs[i] = 1.0f; }
    return t;
}
template <int PV, bool NB>
MVF_DEV void angles(Unit<PV, NB> &t, const NormArgs &a, const Side &s, int u, int64_t b, int64_t l)
{
    if (!t.rot || !s.pos) return;
    const int j = u * PV, per = a.ra / 2, ax = j / per, jj = j - ax * per;
    const int64_t at = b * s.ps + l * a.axes + ax;
    const int64_t p = a.pos64 ? ((const int64_t *)s.pos)[at] : (int64_t)((const int32_t *)s.pos)[at];
#pragma unroll
    for (int i = 0; i < PV; ++i) sincos_turn((uint64_t)p * a.freq[jj + i], t.sn[i], t.cs[i]);
}

template <int N, typename T>
MVF_DEV void load_run(const T *p, float (&v)[N])
{
    const typename Run<T, N>::V x = *(const typename Run<T, N>::U *)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}
template <int N, typename T>
MVF_DEV void store_run(T *p, const float (&v)[N], bool in)
{
    if (!in) return;
    typename Run<T, N>::V x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    *(typename Run<T, N>::U *)p = x;
}
// the unit's 2 PV values of a row, as pairs (v[i], v[PV + i]): two runs of PV channels, each whole inside the row or not there.
// Runs that are not there are loaded from channel 0 and cleared (`ragged`: some lane has one), so that no load waits in a branch
template <int PV, bool NB, typename T>
MVF_DEV void load_unit(const T *row, const Unit<PV, NB> &t, bool ragged, float (&v)[2 * PV])
{
    float r[2][PV];
    load_run<PV>(row + t.c0, r[0]);
    load_run<PV>(row + t.c1, r[1]);
    if (ragged) {
#pragma unroll
        for (int i = 0; i < PV; ++i) {
            r[0][i] = t.live ? r[0][i] : 0.0f;
            r[1][i] = t.live1 ? r[1][i] : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
        v[i] = NB ? r[2 * i / PV][2 * i % PV] : r[0][i];
        v[PV + i] = NB ? r[(2 * i + 1) / PV][(2 * i + 1) % PV] : r[1][i];
    }
}
template <int PV, bool NB, typename T>
MVF_DEV void store_unit(T *row, const Unit<PV, NB> &t, const float (&v)[2 * PV], bool in)
{
    float r[2][PV];
#pragma unroll
    for (int i = 0; i < PV; ++i) {
        r[0][i] = NB ? v[(i & 1) * PV + i / 2] : v[i];
        r[1][i] = NB ? v[((PV + i) & 1) * PV + (PV + i) / 2] : v[PV + i];
    }
    store_run<PV>(row + t.c0, r[0], in && t.live);
    store_run<PV>(row + t.c1, r[1], in && t.live1);
}

template <int CTRL>
MVF_DEV float dpp(float x) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true)); }
MVF_DEV float halves_sum(float x)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
MVF_DEV float rows_sum(float x)
{
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// sums over the aligned groups of `lpr` lanes, in every lane of the group (N of them side by side)
template <int N>
MVF_DEV void group_sum(float (&x)[N], int lpr)
{
#define MVF_EACH(expr)           \
    _Pragma("unroll") for (int k = 0; k < N; ++k) x[k] = (expr)
    if (lpr > 1) MVF_EACH(x[k] + dpp<0xB1>(x[k]));        // quad_perm [1,0,3,2]
    if (lpr > 2) MVF_EACH(x[k] + dpp<0x4E>(x[k]));        // quad_perm [2,3,0,1]
    if (lpr > 4) MVF_EACH(x[k] + dpp<0x141>(x[k]));       // row_half_mirror: the other quad of eight lanes
    if (lpr > 8) MVF_EACH(x[k] + dpp<0x140>(x[k]));       // row_mirror: the other half of sixteen
    if (lpr > 16) MVF_EACH(rows_sum(x[k]));
    if (lpr > 32) MVF_EACH(halves_sum(x[k]));
#undef MVF_EACH
}
// 1 / sqrt(x), also of denormals
MVF_DEV float inv_sqrt(float x)
{
    const bool tiny = x < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(tiny ? x * 0x1p+100f : x);
    return tiny ? r * 0x1p+50f : r;
}

template <typename T, int PV, bool NB>
__global__ void __launch_bounds__(NT) k_qk_norm_fwd(const NormArgs a)
{
    const bool second = blockIdx.x >= a.side[0].blocks;
    const Side &s = a.side[second];
    const int64_t blk = blockIdx.x - (second ? a.side[0].blocks : 0);
    const int u = threadIdx.x & (a.lpr - 1);
    const int64_t g = blk * (NT / a.lpr) + threadIdx.x / a.lpr;
    if (g >= s.groups) return;                                  // whole groups leave together: the butterflies below stay inside one
    const int64_t tok = g / s.chunks;
    const int ch = (int)(g - tok * s.chunks);
    const int64_t b = tok / s.L, l = tok - b * s.L;
    Unit<PV, NB> t = unit_of<PV, NB>(a, u);
    angles(t, a, s, u, b, l);
    float w[2 * PV];
#pragma unroll
    for (int i = 0; i < 2 * PV; ++i) w[i] = 1.0f;
    if (s.w) load_unit<PV, NB>(s.w, t, a.ragged, w);
    const T *x0 = (const T *)s.x + b * s.s[0] + l * s.s[1];
    T *y0 = (T *)s.y + tok * s.H * a.D;
    const int h1 = min(s.H, (ch + 1) * s.hg);
    for (int h0 = ch * s.hg; h0 < h1; h0 += HB) {
        // (heads behind the last are read as the last again and not stored: no branch, so that the loads go out together)
        float v[HB][2 * PV], r[HB];
#pragma unroll
        for (int k = 0; k < HB; ++k) load_unit<PV, NB>(x0 + (int64_t)min(h0 + k, h1 - 1) * s.s[2], t, a.ragged, v[k]);
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            r[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * PV; ++i) r[k] = fmaf(v[k][i], v[k][i], r[k]);
        }
        group_sum(r, a.lpr);
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            const float q = inv_sqrt(fmaf(r[k], a.invD, a.eps));
            float y[2 * PV];
#pragma unroll
            for (int i = 0; i < PV; ++i) {
                const float p = v[k][i] * q * w[i], n = v[k][PV + i] * q * w[PV + i];
                y[i] = fmaf(p, t.cs[i], -(n * t.sn[i]));
                y[PV + i] = fmaf(p, t.sn[i], n * t.cs[i]);
            }
            store_unit<PV, NB>(y0 + (int64_t)(h0 + k) * a.D, t, y, h0 + k < h1);
        }
    }
}

// workgroups walk the groups of a side with a stride; the weight gradient stays in registers until the end
template <typename T, int PV, bool NB>
__global__ void __launch_bounds__(NT) k_qk_norm_bwd(const NormArgs a)
{
    __shared__ float fold[2 * PV][NT];
    const bool second = blockIdx.x >= a.side[0].blocks;
    const Side &s = a.side[second];
    const int64_t blk = blockIdx.x - (second ? a.side[0].blocks : 0);
    const int u = threadIdx.x & (a.lpr - 1), gpb = NT / a.lpr;
    Unit<PV, NB> t = unit_of<PV, NB>(a, u);
    float w[2 * PV], dw[2 * PV];
#pragma unroll
    for (int i = 0; i < 2 * PV; ++i) { w[i] = 1.0f; dw[i] = 0.0f; }
    if (s.w) load_unit<PV, NB>(s.w, t, a.ragged, w);
    for (int64_t g = blk * gpb + threadIdx.x / a.lpr; g < s.groups; g += s.blocks * gpb) {
        const int64_t tok = g / s.chunks;
        const int ch = (int)(g - tok * s.chunks);
        const int64_t b = tok / s.L, l = tok - b * s.L;
        angles(t, a, s, u, b, l);
        const T *x0 = (const T *)s.x + b * s.s[0] + l * s.s[1];
        const T *g0 = (const T *)s.gy + tok * s.H * a.D;
        T *y0 = (T *)s.y + tok * s.H * a.D;
        const int h1 = min(s.H, (ch + 1) * s.hg);
        for (int h0 = ch * s.hg; h0 < h1; h0 += HG) {
            float v[HG][2 * PV], f[HG][2 * PV], sum[2 * HG];
#pragma unroll
            for (int k = 0; k < HG; ++k) {
                const int64_t hk = min(h0 + k, h1 - 1);
                load_unit<PV, NB>(x0 + hk * s.s[2], t, a.ragged, v[k]);
                load_unit<PV, NB>(g0 + hk * a.D, t, a.ragged, f[k]);
            }
#pragma unroll
            for (int k = 0; k < HG; ++k) {
                sum[2 * k] = sum[2 * k + 1] = 0.0f;
#pragma unroll
                for (int i = 0; i < PV; ++i) {                  // u = R(-pos) dy
                    const float e0 = f[k][i], e1 = f[k][PV + i];
                    f[k][i] = fmaf(e0, t.cs[i], e1 * t.sn[i]);
                    f[k][PV + i] = fmaf(e1, t.cs[i], -(e0 * t.sn[i]));
                }
#pragma unroll
                for (int i = 0; i < 2 * PV; ++i) {
                    sum[2 * k] = fmaf(v[k][i], v[k][i], sum[2 * k]);
                    sum[2 * k + 1] = fmaf(f[k][i] * w[i], v[k][i], sum[2 * k + 1]);
                }
            }
            group_sum(sum, a.lpr);
#pragma unroll
            for (int k = 0; k < HG; ++k) {
                const bool in = h0 + k < h1;
                const float r = inv_sqrt(fmaf(sum[2 * k], a.invD, a.eps)), z = sum[2 * k + 1] * r * r * r * a.invD, rw = in ? r : 0.0f;
                float y[2 * PV];
#pragma unroll
                for (int i = 0; i < 2 * PV; ++i) {
                    dw[i] = fmaf(f[k][i] * v[k][i], rw, dw[i]);
                    y[i] = fmaf(f[k][i] * w[i], r, -(v[k][i] * z));
                }
                store_unit<PV, NB>(y0 + (int64_t)(h0 + k) * a.D, t, y, in);
            }
        }
    }
    if (!s.part) return;
#pragma unroll
    for (int i = 0; i < 2 * PV; ++i) fold[i][threadIdx.x] = dw[i];
    __syncthreads();
    if ((int)threadIdx.x < a.lpr && t.live) {
        float *p = s.part + blk * a.D;
#pragma unroll
        for (int i = 0; i < 2 * PV; ++i) {
            float x = 0.0f;
            for (int k = threadIdx.x; k < NT; k += a.lpr) x += fold[i][k];
            if (t.has(i)) p[t.channel(i)] = x;
        }
    }
}

// weight gradients: the partial rows of a side added in order.  grid (16 channels each, side), 16 x 16 lanes
__global__ void __launch_bounds__(NT) k_qk_norm_dw(const float *p0, const float *p1, float *o0, float *o1, int n0, int n1, int D)
{
    __shared__ float fold[16][17];
    const float *p = blockIdx.y ? p1 : p0;
    float *o = blockIdx.y ? o1 : o0;
    const int n = blockIdx.y ? n1 : n0;
    if (!o) return;
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4;
    float x = 0.0f;
    if (c < D) {
#pragma unroll 8
        for (int i = k; i < n; i += 16) x += p[(int64_t)i * D + c];
    }
    fold[k][threadIdx.x & 15] = x;
    __syncthreads();
    if (k == 0 && c < D) {
        float r = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) r += fold[i][threadIdx.x];
        o[c] = r;
    }
}

constexpr int kWant = 1024, kBwdBlocks = 1024;     // workgroups: enough to fill the chip; rows of partial weight gradients

bool bad_desc(const mvf_qk_norm_desc *d)
{
    if (!d || d->B < 0 || d->Lq < 0 || d->Lk < 0 || d->Hq <= 0 || d->Hk <= 0 || d->D <= 0 || d->D > MVF_ATTN_MAX_D) return true;
    if (d->dtype != MVF_DTYPE_F32 && d->dtype != MVF_DTYPE_BF16) return true;
    if (d->rot < 0 || d->rot > d->D || d->axes < 1 || d->axes > 3 || d->rot % (2 * d->axes)) return true;
    if (d->rot && !d->freq) return true;
    const int64_t most = 0x7fffffffLL / 2;
    return (int64_t)d->B * d->Lq * d->Hq > most || (int64_t)d->B * d->Lk * d->Hk > most;
}

// kernel arguments and which variant: returns PV, the longest run of channels (4, 2, 1) that the blocks and the rest are made of; 0 if
// the forward would be too large a launch (the backward walks its rows in fewer workgroups)
int plan(const mvf_qk_norm_desc &d, NormArgs &a, bool bwd)
{
    a = {};
    a.D = d.D; a.axes = d.axes; a.rot = d.rot; a.ra = d.rot / d.axes;
    a.pos64 = d.pos64;
    a.eps = d.eps;
    a.invD = 1.0f / (float)d.D;
    for (int j = 0; j < a.ra / 2; ++j) a.freq[j] = d.freq[j];
    auto fits = [&](int n) { return a.ra / 2 % n == 0 && (d.D - d.rot) % n == 0; };
    const int PV = fits(4) ? 4 : fits(2) ? 2 : 1;
    a.rotu = d.rot / 2 / PV;
    a.units = a.rotu + (d.D - d.rot + 2 * PV - 1) / (2 * PV);
    a.lpr = 1;
    while (a.lpr < a.units) a.lpr *= 2;
    a.ragged = a.units < a.lpr || (d.D - d.rot) % (2 * PV);
    int64_t blocks = 0;
    for (int i = 0; i < 2; ++i) {
        Side &s = a.side[i];
        s.x = i ? d.k : d.q;
        s.w = i ? d.k_weight : d.q_weight;
        s.pos = i ? d.k_pos : d.q_pos;
        s.ps = i ? d.k_pos_stride : d.q_pos_stride;
        for (int j = 0; j < 3; ++j) s.s[j] = i ? d.k_stride[j] : d.q_stride[j];
        s.L = i ? d.Lk : d.Lq;
        s.H = i ? d.Hk : d.Hq;
        const int64_t tokens = s.x ? (int64_t)d.B * s.L : 0, gpb = NT / a.lpr;
        // one group of lanes per token where tokens alone fill the chip, so that a token's angles are formed once; fewer
        // heads per group where they do not
        int64_t c = tokens > 0 ? (kWant * gpb + tokens - 1) / tokens : 1;
        if (c > s.H) c = s.H;
        s.hg = (int)((s.H + c - 1) / c);
        s.chunks = (s.H + s.hg - 1) / s.hg;
        s.groups = tokens * s.chunks;
        s.blocks = (s.groups + gpb - 1) / gpb;
        blocks += s.blocks;
        if (bwd) {                                             // rows of partial weight gradients: half of the workgroups, 256 .. 1,024
            const int64_t most = s.blocks / 2 < 256 ? 256 : s.blocks / 2 > kBwdBlocks ? kBwdBlocks : s.blocks / 2;
            if (s.blocks > most) s.blocks = most;
        }
    }
    return blocks * NT > kMaxThreads ? 0 : PV;
}

#define MVF_NORM_LAUNCH(fn, T, PV)                                                              \
    do {                                                                                        \
        if (d->interleaved) hipLaunchKernelGGL((fn<T, PV, true>), g, b, 0, st, a);              \
        else hipLaunchKernelGGL((fn<T, PV, false>), g, b, 0, st, a);                            \
    } while (0)
#define MVF_NORM_PICK(fn)                                                                       \
    do {                                                                                        \
        if (esz == 4) {                                                                         \
            if (PV == 4) MVF_NORM_LAUNCH(fn, float, 4);                                         \
            else if (PV == 2) MVF_NORM_LAUNCH(fn, float, 2);                                    \
            else MVF_NORM_LAUNCH(fn, float, 1);                                                 \
        } else {                                                                                \
            if (PV == 4) MVF_NORM_LAUNCH(fn, __bf16, 4);                                        \
            else if (PV == 2) MVF_NORM_LAUNCH(fn, __bf16, 2);                                   \
            else MVF_NORM_LAUNCH(fn, __bf16, 1);                                                \
        }                                                                                       \
    } while (0)

}  // namespace

extern "C" {

int mvf_qk_norm_rope_fwd(const mvf_qk_norm_desc *d, void *q_out, void *k_out, void *stream)
{
    if (bad_desc(d)) return (int)hipErrorInvalidValue;
    NormArgs a;
    const int PV = plan(*d, a, false);
    if (!PV || (a.side[0].groups && !q_out) || (a.side[1].groups && !k_out) || (((uintptr_t)q_out | (uintptr_t)k_out) & 15))
        return (int)hipErrorInvalidValue;
    const int64_t blocks = a.side[0].blocks + a.side[1].blocks;
    if (blocks == 0) return 0;
    a.side[0].y = q_out;
    a.side[1].y = k_out;
    hipStream_t st = (hipStream_t)stream;
    const int64_t esz = d->dtype == MVF_DTYPE_F32 ? 4 : 2;
    ProfScope ps(MVF_PROF_QK_NORM_FWD, st, 2 * esz * d->D * d->B * ((d->q ? (int64_t)d->Lq * d->Hq : 0) + (d->k ? (int64_t)d->Lk * d->Hk : 0)));
    const dim3 g((unsigned)blocks), b(NT);
    MVF_NORM_PICK(k_qk_norm_fwd);
    return hip_check_launch();
}

size_t mvf_qk_norm_rope_bwd_workspace_floats(const mvf_qk_norm_desc *d)
{
    if (bad_desc(d)) return 0;
    NormArgs a;
    if (!plan(*d, a, true)) return 0;
    return (size_t)((a.side[0].blocks + a.side[1].blocks) * d->D);
}

int mvf_qk_norm_rope_bwd(const mvf_qk_norm_desc *d, const void *g_q_out, const void *g_k_out, void *g_q, void *g_k,
                         float *g_q_weight, float *g_k_weight, float *workspace, void *stream)
{
    if (bad_desc(d)) return (int)hipErrorInvalidValue;
    NormArgs a;
    const int PV = plan(*d, a, true);
    if (!PV || (a.side[0].groups && (!g_q || !g_q_out)) || (a.side[1].groups && (!g_k || !g_k_out))) return (int)hipErrorInvalidValue;
    if (((uintptr_t)g_q | (uintptr_t)g_k | (uintptr_t)g_q_out | (uintptr_t)g_k_out) & 15) return (int)hipErrorInvalidValue;
    if ((g_q_weight || g_k_weight) && !workspace) return (int)hipErrorInvalidValue;
    const int64_t blocks = a.side[0].blocks + a.side[1].blocks;
    a.side[0].gy = g_q_out; a.side[1].gy = g_k_out;
    a.side[0].y = g_q; a.side[1].y = g_k;
    a.side[0].part = g_q_weight ? workspace : nullptr;
    a.side[1].part = g_k_weight ? workspace + a.side[0].blocks * d->D : nullptr;
    hipStream_t st = (hipStream_t)stream;
    const int64_t esz = d->dtype == MVF_DTYPE_F32 ? 4 : 2;
    ProfScope ps(MVF_PROF_QK_NORM_BWD, st, 3 * esz * d->D * d->B * ((d->q ? (int64_t)d->Lq * d->Hq : 0) + (d->k ? (int64_t)d->Lk * d->Hk : 0)));
    const dim3 g((unsigned)blocks), b(NT);
    if (blocks) {
        MVF_NORM_PICK(k_qk_norm_bwd);
    }
    if (g_q_weight || g_k_weight)
        hipLaunchKernelGGL(k_qk_norm_dw, dim3((unsigned)((d->D + 15) / 16), 2), b, 0, st, a.side[0].part, a.side[1].part, g_q_weight,
                           g_k_weight, (int)a.side[0].blocks, (int)a.side[1].blocks, d->D);
    return hip_check_launch();
}

}  // extern "C"
