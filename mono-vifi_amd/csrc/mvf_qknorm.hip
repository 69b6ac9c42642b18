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
// Angles are exact for any position: a frequency is a 64-bit fixed-point fraction of a turn, so pos * freq modulo one turn is
// one integer product; its top bits give the quadrant and a remainder of at most an eighth of a turn, to which the Taylor
// polynomials of sine (x^9) and cosine (x^10) apply with an error below an fp32 step.  (A product in fp32 loses the angle
// altogether at far positions: half a step of 300,000 is a sixtieth of a radian.)
//
// Bound by memory: 2 passes over the rows forward, 3 backward.  A group of lanes owns a token, so the sines and cosines are
// formed once for all its heads; a lane owns the same pairs of every head, loads them with 8- or 16-byte accesses, and the sum
// of squares is a butterfly over the group.  All arithmetic is fp32; bf16 is rounded once, at the store.
#include "mvf_common.hpp"

using namespace mvf;

namespace {

constexpr int NT = 256;
constexpr int HB = 4;             // heads in flight per lane

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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
    int pos64;
    float eps;
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
    int c0, c1;
    bool live, rot;
    float sn[PV], cs[PV];
    MVF_DEV int channel(int i) const { return NB ? (i < PV ? c0 + 2 * i : c0 + 2 * (i - PV) + 1) : (i < PV ? c0 + i : c1 + i - PV); }
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
        t.c1 = t.c0 + per;
    } else {
        t.c0 = a.rot + (u - a.rotu) * 2 * PV;
        t.c1 = t.c0 + PV;
    }
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

template <int N>
MVF_DEV void load_run(const float *p, float *v)
{
    static_assert(N == 4, "");
    const f32x4 x = *(const f32x4 *)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x[i];
}
template <int N>
MVF_DEV void load_run(const __bf16 *p, float *v)
{
    static_assert(N == 4, "");
    const bf16x4 x = *(const bf16x4 *)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}
MVF_DEV void store_run(float *p, const float *v) { *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]}; }
MVF_DEV void store_run(__bf16 *p, const float *v)
{
    bf16x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (__bf16)v[i];
    *(bf16x4 *)p = x;
}

// the unit's 2 PV values of a row, as pairs (v[i], v[PV + i])
template <int PV, bool NB, typename T>
MVF_DEV void load_unit(const T *row, const Unit<PV, NB> &t, int D, float (&v)[2 * PV])
{
    if constexpr (PV == 1) {
        v[0] = t.live && t.channel(0) < D ? (float)row[t.channel(0)] : 0.0f;
        v[1] = t.live && t.channel(1) < D ? (float)row[t.channel(1)] : 0.0f;
    } else {
        float a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
        if (t.live) {
            load_run<4>(row + t.c0, a);
            load_run<4>(row + (NB ? t.c0 + 4 : t.c1), b);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = NB ? (i < 2 ? a[2 * i & 3] : b[2 * i & 3]) : a[i];
            v[4 + i] = NB ? (i < 2 ? a[(2 * i + 1) & 3] : b[(2 * i + 1) & 3]) : b[i];
        }
    }
}
template <int PV, bool NB, typename T>
MVF_DEV void store_unit(T *row, const Unit<PV, NB> &t, int D, const float (&v)[2 * PV])
{
    if (!t.live) return;
    if constexpr (PV == 1) {
        if (t.channel(0) < D) row[t.channel(0)] = (T)v[0];
        if (t.channel(1) < D) row[t.channel(1)] = (T)v[1];
    } else if constexpr (NB) {
        const float a[4] = {v[0], v[4], v[1], v[5]}, b[4] = {v[2], v[6], v[3], v[7]};
        store_run(row + t.c0, a);
        store_run(row + t.c0 + 4, b);
    } else {
        const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
        store_run(row + t.c0, a);
        store_run(row + t.c1, b);
    }
}
MVF_DEV float group_sum(float x, int lpr)
{
    for (int m = lpr >> 1; m > 0; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
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
    if (s.w) load_unit<PV, NB>(s.w, t, a.D, w);
    const T *x0 = (const T *)s.x + b * s.s[0] + l * s.s[1];
    T *y0 = (T *)s.y + tok * s.H * a.D;
    const int h1 = min(s.H, (ch + 1) * s.hg);
    for (int h0 = ch * s.hg; h0 < h1; h0 += HB) {
        float v[HB][2 * PV];
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            if (h0 + k < h1) {
                load_unit<PV, NB>(x0 + (int64_t)(h0 + k) * s.s[2], t, a.D, v[k]);
            } else {
#pragma unroll
                for (int i = 0; i < 2 * PV; ++i) v[k][i] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            // (the butterfly runs for heads behind the last too, on zeros: no branch, so that the rows stay in registers)
            float q = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * PV; ++i) q = fmaf(v[k][i], v[k][i], q);
            const float r = 1.0f / sqrtf(group_sum(q, a.lpr) / (float)a.D + a.eps);
            float y[2 * PV];
#pragma unroll
            for (int i = 0; i < PV; ++i) {
                const float p = v[k][i] * r * w[i], n = v[k][PV + i] * r * w[PV + i];
                y[i] = fmaf(p, t.cs[i], -(n * t.sn[i]));
                y[PV + i] = fmaf(p, t.sn[i], n * t.cs[i]);
            }
            if (h0 + k < h1) store_unit<PV, NB>(y0 + (int64_t)(h0 + k) * a.D, t, a.D, y);
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
    if (s.w) load_unit<PV, NB>(s.w, t, a.D, w);
    for (int64_t g = blk * gpb + threadIdx.x / a.lpr; g < s.groups; g += s.blocks * gpb) {
        const int64_t tok = g / s.chunks;
        const int ch = (int)(g - tok * s.chunks);
        const int64_t b = tok / s.L, l = tok - b * s.L;
        angles(t, a, s, u, b, l);
        const T *x0 = (const T *)s.x + b * s.s[0] + l * s.s[1];
        const T *g0 = (const T *)s.gy + tok * s.H * a.D;
        T *y0 = (T *)s.y + tok * s.H * a.D;
        const int h1 = min(s.H, (ch + 1) * s.hg);
        for (int h0 = ch * s.hg; h0 < h1; h0 += HB) {
            float v[HB][2 * PV], e[HB][2 * PV];
#pragma unroll
            for (int k = 0; k < HB; ++k) {
                if (h0 + k < h1) {
                    load_unit<PV, NB>(x0 + (int64_t)(h0 + k) * s.s[2], t, a.D, v[k]);
                    load_unit<PV, NB>(g0 + (int64_t)(h0 + k) * a.D, t, a.D, e[k]);
                } else {
#pragma unroll
                    for (int i = 0; i < 2 * PV; ++i) v[k][i] = e[k][i] = 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < HB; ++k) {
                float q = 0.0f, d = 0.0f;
                float f[2 * PV];                                // u = R(-pos) dy
#pragma unroll
                for (int i = 0; i < PV; ++i) {
                    f[i] = fmaf(e[k][i], t.cs[i], e[k][PV + i] * t.sn[i]);
                    f[PV + i] = fmaf(e[k][PV + i], t.cs[i], -(e[k][i] * t.sn[i]));
                }
#pragma unroll
                for (int i = 0; i < 2 * PV; ++i) {
                    q = fmaf(v[k][i], v[k][i], q);
                    d = fmaf(f[i] * w[i], v[k][i], d);
                }
                q = group_sum(q, a.lpr);
                d = group_sum(d, a.lpr);
                const float r = 1.0f / sqrtf(q / (float)a.D + a.eps);
                const float z = d * r * r * r / (float)a.D;
                float y[2 * PV];
#pragma unroll
                for (int i = 0; i < 2 * PV; ++i) {
                    dw[i] = fmaf(f[i] * v[k][i], r, dw[i]);
                    y[i] = fmaf(f[i] * w[i], r, -(v[k][i] * z));
                }
                if (h0 + k < h1) store_unit<PV, NB>(y0 + (int64_t)(h0 + k) * a.D, t, a.D, y);
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
            const int c = t.channel(i);
            if (c < a.D) p[c] = x;
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
    if (c < D)
        for (int i = k; i < n; i += 16) x += p[(int64_t)i * D + c];
    fold[k][threadIdx.x & 15] = x;
    __syncthreads();
    if (k == 0 && c < D) {
        float r = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) r += fold[i][threadIdx.x];
        o[c] = r;
    }
}

constexpr int kWant = 2048, kBwdBlocks = 1024;     // workgroups: enough to fill the chip; rows of partial weight gradients

bool bad_desc(const mvf_qk_norm_desc *d)
{
    if (!d || d->B < 0 || d->Lq < 0 || d->Lk < 0 || d->Hq <= 0 || d->Hk <= 0 || d->D <= 0 || d->D > MVF_ATTN_MAX_D) return true;
    if (d->dtype != MVF_DTYPE_F32 && d->dtype != MVF_DTYPE_BF16) return true;
    if (d->rot < 0 || d->rot > d->D || d->axes < 1 || d->axes > 3 || d->rot % (2 * d->axes)) return true;
    if (d->rot && !d->freq) return true;
    const int64_t most = 0x7fffffffLL / 2;
    return (int64_t)d->B * d->Lq * d->Hq > most || (int64_t)d->B * d->Lk * d->Hk > most;
}

// kernel arguments and which variant: returns PV (4 where every access of a unit is an aligned run of four channels, else 1)
int plan(const mvf_qk_norm_desc &d, NormArgs &a, bool bwd)
{
    a = {};
    a.D = d.D; a.axes = d.axes; a.rot = d.rot; a.ra = d.rot / d.axes;
    a.pos64 = d.pos64;
    a.eps = d.eps;
    for (int j = 0; j < a.ra / 2; ++j) a.freq[j] = d.freq[j];
    bool wide = a.ra % 8 == 0 && (d.D - d.rot) % 8 == 0;
    for (int i = 0; i < 3; ++i) wide = wide && d.q_stride[i] % 4 == 0 && d.k_stride[i] % 4 == 0;
    const uintptr_t bits = (uintptr_t)d.q | (uintptr_t)d.k | (uintptr_t)d.q_weight | (uintptr_t)d.k_weight;
    wide = wide && !(bits & 15);
    const int PV = wide ? 4 : 1;
    a.rotu = d.rot / 2 / PV;
    a.units = a.rotu + (d.D - d.rot + 2 * PV - 1) / (2 * PV);
    a.lpr = 1;
    while (a.lpr < a.units) a.lpr *= 2;
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
        if (bwd && s.blocks > kBwdBlocks) s.blocks = kBwdBlocks;
    }
    return PV;
}

#define MVF_NORM_LAUNCH(fn, T, PV)                                                              \
    do {                                                                                        \
        if (d->interleaved) hipLaunchKernelGGL((fn<T, PV, true>), g, b, 0, st, a);              \
        else hipLaunchKernelGGL((fn<T, PV, false>), g, b, 0, st, a);                            \
    } while (0)
#define MVF_NORM_PICK(fn)                                                                       \
    do {                                                                                        \
        if (esz == 4 && PV == 4) MVF_NORM_LAUNCH(fn, float, 4);                                 \
        else if (esz == 4) MVF_NORM_LAUNCH(fn, float, 1);                                       \
        else if (PV == 4) MVF_NORM_LAUNCH(fn, __bf16, 4);                                       \
        else MVF_NORM_LAUNCH(fn, __bf16, 1);                                                    \
    } while (0)

}  // namespace

extern "C" {

int mvf_qk_norm_rope_fwd(const mvf_qk_norm_desc *d, void *q_out, void *k_out, void *stream)
{
    if (bad_desc(d)) return (int)hipErrorInvalidValue;
    NormArgs a;
    const int PV = plan(*d, a, false);
    if ((a.side[0].groups && !q_out) || (a.side[1].groups && !k_out) || (((uintptr_t)q_out | (uintptr_t)k_out) & 15))
        return (int)hipErrorInvalidValue;
    const int64_t blocks = a.side[0].blocks + a.side[1].blocks;
    if (blocks == 0) return 0;
    if (blocks > 0x7fffffffLL) return (int)hipErrorInvalidValue;
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
    plan(*d, a, true);
    return (size_t)((a.side[0].blocks + a.side[1].blocks) * d->D);
}

int mvf_qk_norm_rope_bwd(const mvf_qk_norm_desc *d, const void *g_q_out, const void *g_k_out, void *g_q, void *g_k,
                         float *g_q_weight, float *g_k_weight, float *workspace, void *stream)
{
    if (bad_desc(d)) return (int)hipErrorInvalidValue;
    NormArgs a;
    const int PV = plan(*d, a, true);
    if ((a.side[0].groups && (!g_q || !g_q_out)) || (a.side[1].groups && (!g_k || !g_k_out))) return (int)hipErrorInvalidValue;
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
