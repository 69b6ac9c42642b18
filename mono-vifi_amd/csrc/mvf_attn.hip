// mvf_attn.hip -- cross attention of the tokens of one frame to the tokens of others: forward and backward.
//
//     o[b,i,h] = sum_j P[i,j] v[b,j,h/G],  P[i,:] = softmax_j(scale * q[b,i,h] . k[b,j,h/G]) over the states j that count
//
// with G = Hq / Hk query heads reading one head of keys and values, kv_lens[b] states per sequence and a byte mask of
// states.  A state that does not count contributes nothing whatever its memory holds (it is staged as zeros, its score is
// -inf); a query no state counts for gets zeros, and zero gradients.
//
// The scores never reach memory.  A wave owns 32 query rows (row r = i * G + g: the G heads that share a head of keys are
// rows of the same tile, so one staged tile serves them all) and walks the states in tiles, keeping the running maximum m,
// the sum l and the output tile in registers:
//     S^T = K Q^T (32 x 32 x 16 matrix instructions: a lane holds ONE query, 16 of the 32 states of a tile),
//     m' = max(m, max S), P^T = exp2(c S^T - c m'), l' = l exp2(c m - c m') + sum P,  O^T = O^T exp2(c m - c m') + V^T P^T
// with c = scale * log2(e).  Computing the TRANSPOSED products keeps the softmax of a query inside two lanes (lane, lane ^ 32)
// and makes the accumulator of S^T directly the right operand of V^T P^T: the order in which a lane holds the states of a
// tile is a permutation of the reduction index, and V is read from LDS in the same permutation (ds_read_b64_tr_b16: four
// states of one channel per lane), so P never moves between lanes.
//
// Types.  Everything the matrix units multiply is bf16; sums are fp32.  bf16 inputs are one plane.  What becomes an operand of a second
// product (P before V^T P and P^T do, dS before dq and dk) is two planes, 2^-16 of a term, where that matters or is free (kSmall, below),
// else one, rounded: 2^-8 of a term at most.  The results of one plane (large inference outputs, dk and dv) are 2.3e-3 - 2.4e-3 from the
// 64-bit ones (relative 2-norm), those of two 1.7e-3, which is the rounding of the result itself.  fp32 inputs are three
// (x = x0 + x1 + x2, each the leading 8 significand bits of what the previous left: exact), a product the six terms of
// order <= 2: relative error below 2^-21 per product, and still 2.6 x the rate of the fp32 matrix instructions (6 x 32 cycles
// against 8 x 64 for a 32 x 32 x 16 product).
//
// Compiled without contraction (the library's flag); fused multiply-adds are written out.
#include "mvf_common.hpp"

using namespace mvf;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256;            // four waves
constexpr int PADE = 8;            // bf16 elements appended to an LDS row: rows 16 bytes apart modulo 128
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Staged tiles: two buffers (one barrier per tile) for one plane, one buffer (two barriers) for three, whose tiles would halve
// the number of resident workgroups (1,920 x 3,840 x 32 fp32 forward: 264 against 285 us)
constexpr int buffers(int NP) { return NP == 1 ? 2 : 1; }

#define LDS_PTR(T) __attribute__((address_space(3))) T *

// ------------------------------------------------------------------------------------------------- planes
template <int NP>
struct Frag {
    bf16x8 p[NP];
};
template <int NP>
struct Elem;
template <>
struct Elem<1> {
    typedef __bf16 T;
};
template <>
struct Elem<3> {
    typedef float T;
};

MVF_DEV float trunc_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
MVF_DEV short top16(float x) { return (short)(__float_as_uint(x) >> 16); }

// eight fp32 values -> NP planes of bf16.  One plane rounds to nearest even (half a step, 2^-8 of the value); three planes
// cut, so that every remainder is exact.  (An infinity leaves a NaN behind: what it takes part in becomes NaN.)
template <int NP>
MVF_DEV Frag<NP> split8(const float (&x)[8])
{
    Frag<NP> f;
    if constexpr (NP == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f.p[0][e] = (__bf16)x[e];
    } else {
        s16x8 a, b, c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float hi = trunc_bf16(x[e]);
            const float r1 = x[e] - hi;
            const float mid = trunc_bf16(r1);
            a[e] = top16(hi);
            b[e] = top16(mid);
            c[e] = top16(r1 - mid);
        }
        f.p[0] = __builtin_bit_cast(bf16x8, a);
        f.p[1] = __builtin_bit_cast(bf16x8, b);
        f.p[2] = __builtin_bit_cast(bf16x8, c);
    }
    return f;
}

// eight fp32 values as two planes: the leading 8 significand bits (cut), and what they leave, rounded to 8 bits.  P: of probabilities, whose
// second plane is never zero -- an infinite value of a state that counts has to come out as an infinity, and 0 x inf is none
template <bool P>
MVF_DEV void split8(const float (&x)[8], Frag<1> &hi, Frag<1> &lo)
{
    s16x8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        a[e] = top16(x[e]);
        const float rest = x[e] - trunc_bf16(x[e]);
        lo.p[0][e] = (__bf16)(P ? fmaxf(rest, 0x1p-126f) : rest);
    }
    hi.p[0] = __builtin_bit_cast(bf16x8, a);
}

// c += a b; the small terms of the three-plane product first
template <int NP>
MVF_DEV f32x16 mma(const Frag<NP> &a, const Frag<NP> &b, f32x16 c)
{
    if constexpr (NP == 3) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

// The same bits as mma(b, a) with rows and columns exchanged: the terms in the other order.
template <int NP>
MVF_DEV f32x16 mma_exchanged(const Frag<NP> &a, const Frag<NP> &b, f32x16 c)
{
    if constexpr (NP == 3) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

// the same for 16 x 16 tiles: 32 channels or states per product
template <int NP>
MVF_DEV f32x4 mma(const Frag<NP> &a, const Frag<NP> &b, f32x4 c)
{
    if constexpr (NP == 3) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[2], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

constexpr uint32_t kNowhere = 0x80000000u;       // a byte offset behind every buffer: loads give zeros

// eight channels of a row as loaded
template <int NP>
struct Raw;
template <>
struct Raw<1> {
    bf16x8 x;
    MVF_DEV void zero() { x = bf16x8{}; }
    MVF_DEV void load(__amdgpu_buffer_rsrc_t rs, uint32_t at, bool) { x = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0)); }
    MVF_DEV Frag<1> frag() const { return Frag<1>{{x}}; }
    MVF_DEV Frag<1> frag_scaled(float) const { return frag(); }
};
template <>
struct Raw<3> {
    f32x4 a, b;
    MVF_DEV void zero() { a = b = f32x4{}; }
    MVF_DEV void load(__amdgpu_buffer_rsrc_t rs, uint32_t at, bool more)      // more: the row has the last four channels too
    {
        a = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0));
        b = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, more ? at + 16 : kNowhere, 0, 0));
    }
    MVF_DEV Frag<3> frag() const
    {
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return split8<3>(x);
    }
    MVF_DEV Frag<3> frag_scaled(float f) const
    {
        const float x[8] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f, b[0] * f, b[1] * f, b[2] * f, b[3] * f};
        return split8<3>(x);
    }
};
// The factor c of the exponent: three planes take it into q before it is cut, one rounding of fp32 among those of the products, so
// that the scores come out of the matrix units ready; one plane would round the product to bf16.  In three planes all kernels
// of a training step form the same bits of a score, by the same products in the same order: a score of 150 rounds by 8e-6, and a
// probability whose exponent and reference rounded apart would be off by that (dv at scores of 150: 1.2e-5 of the result).
template <int NP>
MVF_DEV float exponent(float s, float c, float minus) { return NP == 3 ? s + minus : fmaf(s, c, minus); }
// channels d0 .. d0 + 7 of a row of D channels (zeros behind D, or if the row is not `live`); `wide`: rows are 16-byte aligned
// and whole 16-byte runs
MVF_DEV Raw<1> load8(const __bf16 *row, int d0, int D, bool wide, bool live)
{
    Raw<1> r;
    r.zero();
    if (!live) return r;
    if (wide) {
        if (d0 < D) r.x = *(const bf16x8 *)(row + d0);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (d0 + e < D) r.x[e] = row[d0 + e];
    }
    return r;
}
MVF_DEV Raw<3> load8(const float *row, int d0, int D, bool wide, bool live)
{
    Raw<3> r;
    r.zero();
    if (!live) return r;
    if (wide) {
        if (d0 < D) {
            r.a = *(const f32x4 *)(row + d0);
            if (d0 + 4 < D) r.b = *(const f32x4 *)(row + d0 + 4);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (d0 + e < D) r.a[e] = row[d0 + e];
            if (d0 + 4 + e < D) r.b[e] = row[d0 + 4 + e];
        }
    }
    return r;
}
// acc + the dot product of two rows' channels
MVF_DEV float dot8(const Raw<1> &x, const Raw<1> &y, float acc)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = fmaf((float)x.x[e], (float)y.x[e], acc);
    return acc;
}
MVF_DEV float dot8(const Raw<3> &x, const Raw<3> &y, float acc)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = fmaf(x.b[e], y.b[e], fmaf(x.a[e], y.a[e], acc));
    return acc;
}
template <int NP>
MVF_DEV Frag<NP> load_frag(const typename Elem<NP>::T *row, int d0, int D, bool wide, bool live)
{
    return load8(row, d0, D, wide, live).frag();
}

// ------------------------------------------------------------------------------------------------- LDS tiles
// a tile of ROWS x DP values: NP planes of [ROWS][DP + PADE] bf16
template <int NP, int ROWS, int DP>
struct Tile {
    static constexpr int LD = DP + PADE, PLANE = ROWS * LD;
    short v[NP * PLANE];

    // one 8-channel chunk
    MVF_DEV void put(int row, int chunk, const Frag<NP> &f)
    {
#pragma unroll
        for (int p = 0; p < NP; ++p) *(bf16x8 *)&v[p * PLANE + row * LD + chunk * 8] = f.p[p];
    }
    // left operand whose rows are the tile's rows, reduced over 16 channels: row r0 + (lane & 31), channels k0 + 8 (lane >> 5) + e
    MVF_DEV Frag<NP> rows(int r0, int k0, int lane) const
    {
        Frag<NP> f;
#pragma unroll
        for (int p = 0; p < NP; ++p) f.p[p] = *(const bf16x8 *)&v[p * PLANE + (r0 + (lane & 31)) * LD + k0 + 8 * (lane >> 5)];
        return f;
    }
    // left operand whose rows are channels d0 + (lane & 31), reduced over the 16 rows r0 .. r0 + 15 in the order an
    // accumulator holds them: element e of lane half h is row r0 + 4h + (e & 3) + 8 (e >> 2).  The transposing read hands
    // lane t of a group of 16 the four rows of column t; lane t supplies the address of row t / 4, columns 4 (t & 3) ..
    MVF_DEV Frag<NP> cols(int d0, int r0, int lane) const
    {
        const int row = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2), col = d0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        Frag<NP> f;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const short *a = &v[p * PLANE + row * LD + col];
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))a);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(a + 8 * LD));
            s16x8 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = lo[e]; x[4 + e] = hi[e]; }
            f.p[p] = __builtin_bit_cast(bf16x8, x);
        }
        return f;
    }
    // the same of 16 channels d0 + (lane & 15), reduced over the first 32 rows in the order two 16-row accumulators hold them:
    // element e of lane quarter g is row 4 g + (e & 3) + 16 (e >> 2)
    MVF_DEV Frag<NP> cols16(int d0, int lane) const
    {
        const int row = 4 * (lane >> 4) + ((lane & 15) >> 2), col = d0 + 4 * (lane & 3);
        Frag<NP> f;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const short *a = &v[p * PLANE + row * LD + col];
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))a);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(a + 16 * LD));
            s16x8 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = lo[e]; x[4 + e] = hi[e]; }
            f.p[p] = __builtin_bit_cast(bf16x8, x);
        }
        return f;
    }
};

// ------------------------------------------------------------------------------------------------- arguments
struct AttnArgs {
    const void *q, *k, *v, *o, *go;
    void *out, *low, *dq, *dk, *dv;           // low: what the rounding of out left (bf16 training), or null
    float *lse, *inv, *delta, *part, *part2;  // inv: 1 / the softmax sum (fp32), or null: in lse
    const uint8_t *mask;
    const int32_t *lens;
    int64_t qs[3], ks[3], vs[3], ms[2];       // batch, token, head strides in elements; mask: batch, state
    int B, Lq, Lk, Hq, Hk, D, G, R;           // R = Lq * G rows per (batch, key head)
    int tiles, splits, per;                   // row or state tiles of a block row, parts of the reduction, reduction tiles per part
    int wide;
    float scale, c;                           // c = scale * log2(e)
};

// Consecutive workgroups go to consecutive XCDs, whose L2s do not share: give every XCD one contiguous run of the
// (sequence, head)-major order, so that the tiles that read the same keys and values find them in one L2.
MVF_DEV int xcd_run(int bid, int n)
{
    const int q = n >> 3, r = n & 7, x = bid & 7, y = bid >> 3;
    return x * q + min(x, r) + y;
}

// Workgroups that share a CU (256 apart in dispatch order) run at different wave priorities: waves of equal priority take turns
// in the matrix units, finish together and then wait together for the vector units; unequal ones fall out of step.
// (1,920 x 3,840 x 32 fp32 backward: 842 -> 815 us; the others 0 - 2 %.)
MVF_DEV void stagger()
{
    switch ((blockIdx.x >> 8) & 3) {
    case 1: __builtin_amdgcn_s_setprio(1); break;
    case 2: __builtin_amdgcn_s_setprio(2); break;
    case 3: __builtin_amdgcn_s_setprio(3); break;
    default: break;
    }
}

MVF_DEV int64_t row_off(const int64_t (&s)[3], int b, int r, int hk, int G)
{
    const int i = G == 1 ? r : r / G, g = G == 1 ? 0 : r - i * G;
    return (int64_t)b * s[0] + (int64_t)i * s[1] + (int64_t)(hk * G + g) * s[2];
}
MVF_DEV int64_t dense_row(int b, int r, int hk, const AttnArgs &a)       // row of a contiguous [B, Lq, Hq, D]
{
    const int i = a.G == 1 ? r : r / a.G, g = a.G == 1 ? 0 : r - i * a.G;
    return (((int64_t)b * a.Lq + i) * a.Hq + hk * a.G + g) * a.D;
}
MVF_DEV int states_of(const AttnArgs &a, int b)
{
    return a.lens ? max(0, min(a.lens[b], a.Lk)) : a.Lk;
}
// which of the 64 states from j0 on count, as a bit each (the same in every lane)
MVF_DEV uint64_t live_states(const AttnArgs &a, int b, int j0, int n, int lane)
{
    const int j = j0 + lane;
    bool ok = j < n;
    if (ok && a.mask) ok = a.mask[(int64_t)b * a.ms[0] + (int64_t)j * a.ms[1]] != 0;
    return __ballot(ok);
}

// This lane's chunks of a tile in flight: fetch() starts the loads of the rows, which lie off(row) elements behind `base` (the
// same in every lane; rows that are not valid(row) become zeros), commit() puts them into the tile.  The loads of a tile are
// issued before the products of the one before it.  WIDE: 16-byte buffer loads, whose bounds check makes the zeros -- no branch,
// so that all of a tile's loads are in flight at once; the host has checked that 32-bit byte offsets reach the rows of a tile.
template <int NP, int ROWS, int DP, bool WIDE>
struct Flight {
    typedef typename Elem<NP>::T T;
    static constexpr int CPR = DP / 8, CHUNKS = ROWS * CPR, N = (CHUNKS + NT - 1) / NT;
    Raw<NP> r[N];
    static MVF_DEV int row_of(int i) { return (i * NT + (int)threadIdx.x) / CPR; }
    static MVF_DEV int chan_of(int i) { return ((i * NT + (int)threadIdx.x) % CPR) * 8; }
    // `all`: every row is valid (the same in every lane)
    template <typename V, typename F>
    MVF_DEV void fetch(const T *base, int D, bool all, V valid, F off)
    {
        if constexpr (WIDE) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)uniform_ptr(base), (short)0, 0x7fffffff, 0x00027000);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = (CHUNKS % NT == 0 || i * NT + threadIdx.x < CHUNKS) && chan_of(i) < D;
                uint32_t at = in ? (uint32_t)(off(i, row_of(i)) + chan_of(i)) * (uint32_t)sizeof(T) : kNowhere;
                if (!all && !valid(row_of(i))) at = kNowhere;
                r[i].load(rs, at, chan_of(i) + 4 < D);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = (CHUNKS % NT == 0 || i * NT + threadIdx.x < CHUNKS) && valid(row_of(i));
                r[i] = load8(base + (in ? off(i, row_of(i)) : 0), chan_of(i), D, false, in);
            }
        }
    }
    MVF_DEV void commit(Tile<NP, ROWS, DP> &t) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (CHUNKS % NT == 0 || i * NT + threadIdx.x < CHUNKS) t.put(row_of(i), chan_of(i) / 8, r[i].frag());
    }
    // the same, rows times f(i) (three planes)
    template <typename F>
    MVF_DEV void commit(Tile<NP, ROWS, DP> &t, F f) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (CHUNKS % NT == 0 || i * NT + threadIdx.x < CHUNKS) t.put(row_of(i), chan_of(i) / 8, r[i].frag_scaled(f(i)));
    }
};
template <bool WIDE>
struct Stride;                    // a stride, as wide as the offsets within a tile have to be
template <>
struct Stride<true> {
    typedef int T;
};
template <>
struct Stride<false> {
    typedef int64_t T;
};

// Products whose left operands come from LDS: load(i) is issued AHEAD steps before mul(i, operand), and the order of the two
// kinds is pinned (other instructions may cross), so that a wave waits for LDS once and not once per product.
template <int NP>
constexpr int kAhead = NP == 1 ? 4 : 1;
#define MVF_PIN() __builtin_amdgcn_sched_barrier(0x2 | 0x4 | 0x10 | 0x200 | 0x400)     /* may cross: VALU, SALU, VMEM, LDS writes, transcendentals */
template <int NP, int N, typename L, typename M>
MVF_DEV void stream(L load, M mul)
{
    constexpr int A = kAhead<NP> < N ? kAhead<NP> : N;
    Frag<NP> f[N];
#pragma unroll
    for (int i = 0; i < A; ++i) f[i] = load(i);
    MVF_PIN();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i + A < N) f[i + A] = load(i + A);
        MVF_PIN();
        mul(i, f[i]);
        MVF_PIN();
    }
}

// What the backward needs of a row's softmax.  lse: the reference of its exponentials, and 1 / their sum beside it (fp32) -- or both in one
// number, the log2 of the sum: in fp32 that rounds at the size of the scores, the same way for all of the row (2^-17 of P at scores of
// 150), where m is a score and s - m is exact where it matters.  INFINITY: no state counts, every exponential is zero.
template <bool F32>
MVF_DEV void store_softmax(const AttnArgs &a, int64_t at, float m, float l)
{
    const bool apart = F32 && a.inv;
    a.lse[at] = l == 0.0f ? INFINITY : apart ? m : m + __builtin_amdgcn_logf(l);
    if (apart) a.inv[at] = l == 0.0f ? 1.0f : 1.0f / l;
}

// The tiles of states a workgroup walks: [j, end) in steps of BK, those without a state that counts left out.  The same in
// every lane of the workgroup.
template <int BK>
struct Walk {
    int j, end, n, b, lane;
    uint64_t bits;
    static constexpr uint64_t kFull = BK == 64 ? ~0ull : (1ull << (BK & 63)) - 1;
    MVF_DEV Walk(const AttnArgs &a, int b_, int part, int lane_) : b(b_), lane(lane_), bits(0)
    {
        n = states_of(a, b);
        j = part * a.per * BK;
        end = (int)min((int64_t)n, (int64_t)(part + 1) * a.per * BK);
        settle(a);
    }
    MVF_DEV bool live() const { return j < end; }
    MVF_DEV void next(const AttnArgs &a)
    {
        j += BK;
        settle(a);
    }
    MVF_DEV void settle(const AttnArgs &a)
    {
        for (; j < end; j += BK) {
            bits = live_states(a, b, j, n, lane) & kFull;
            if (bits) return;
        }
    }
};

MVF_DEV float other_half_max(float x)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
MVF_DEV float other_half_sum(float x)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// and of the lanes 16 apart
MVF_DEV float other_row_max(float x)
{
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
MVF_DEV float other_row_sum(float x)
{
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// state (or row) of accumulator element r of lane half h within a 32-tile
MVF_DEV constexpr int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// elements 8 s .. 8 s + 7 of an accumulator as the right operand of a product reduced over the rows r0 = 16 s .. of the tile
template <int NP>
MVF_DEV Frag<NP> acc_frag(const f32x16 &x, int s)
{
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[8 * s + e];
    return split8<NP>(y);
}
template <bool P>
MVF_DEV void acc_frag(const f32x16 &x, int s, Frag<1> &hi, Frag<1> &lo)
{
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[8 * s + e];
    split8<P>(y, hi, lo);
}

// what rounding to bf16 leaves of a value
MVF_DEV float rest_bf16(float x) { return x - (float)(__bf16)x; }

// four consecutive channels d .. d + 3 of a row
MVF_DEV void store4(float *row, int d, int D, bool wide, float a, float b, float c, float e)
{
    if (wide && d < D) { *(f32x4 *)(row + d) = f32x4{a, b, c, e}; return; }
    const float x[4] = {a, b, c, e};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d + i < D) row[d + i] = x[i];
}
MVF_DEV void store4(__bf16 *row, int d, int D, bool wide, float a, float b, float c, float e)
{
    const float x[4] = {a, b, c, e};
    if (wide && d < D) {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        bf16x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (__bf16)x[i];
        *(bf16x4 *)(row + d) = y;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d + i < D) row[d + i] = (__bf16)x[i];
}
// what the rounding of x f to bf16 left, rounded itself
template <typename T>
MVF_DEV void store_rest(T *row, int d, int D, const float (&x)[4], float f)
{
    store4(row, d, D, (D & 3) == 0, rest_bf16(x[0] * f), rest_bf16(x[1] * f), rest_bf16(x[2] * f), rest_bf16(x[3] * f));
}
// accumulator tiles (channel rows, this lane's column) -> a row of D channels, scaled
template <int DT, typename T>
MVF_DEV void store_cols(T *row, const f32x16 (&acc)[DT], float f, int D, bool wide, int h)
{
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            store4(row, 32 * t + 8 * i + 4 * h, D, wide, acc[t][4 * i] * f, acc[t][4 * i + 1] * f, acc[t][4 * i + 2] * f,
                   acc[t][4 * i + 3] * f);
}

template <int DT, typename T>
MVF_DEV void store_cols_rest(T *row, const f32x16 (&acc)[DT], float f, int D, int h)
{
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x[4] = {acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]};
            store_rest(row, 32 * t + 8 * i + 4 * h, D, x, f);
        }
}

// acc[d] += (32 channels d of the tile's rows r0 .. r0 + 31)^T x.  TWO: x as two planes of bf16 instead of one (P: of probabilities).  NP == 3: the products of a tile are summed on their own and
// then added to the running sum, so that its roundings are one per tile and not one per matrix instruction (3,840 states:
// error 5e-6 -> 1e-6 of the result).
template <int NP, bool TWO, bool P, int DT, int ROWS, int DP>
MVF_DEV void accumulate(f32x16 (&acc)[DT], const Tile<NP, ROWS, DP> &t, int r0, const f32x16 &x, int lane)
{
    static_assert(NP == 1 || !TWO, "");
    if constexpr (TWO) {
        Frag<1> hi[2], lo[2];
        acc_frag<P>(x, 0, hi[0], lo[0]);
        acc_frag<P>(x, 1, hi[1], lo[1]);
        stream<NP, 2 * DT>([&](int i) { return t.cols(32 * (i % DT), r0 + 16 * (i / DT), lane); },
                           [&](int i, const Frag<NP> &f) { acc[i % DT] = mma(f, hi[i / DT], mma(f, lo[i / DT], acc[i % DT])); });
        return;
    }
    const Frag<NP> xf[2] = {acc_frag<NP>(x, 0), acc_frag<NP>(x, 1)};
    if constexpr (NP == 1) {
        stream<NP, 2 * DT>([&](int i) { return t.cols(32 * (i % DT), r0 + 16 * (i / DT), lane); },
                           [&](int i, const Frag<NP> &f) { acc[i % DT] = mma(f, xf[i / DT], acc[i % DT]); });
    } else {
        f32x16 y;
        stream<NP, 2 * DT>([&](int i) { return t.cols(32 * (i / 2), r0 + 16 * (i % 2), lane); },
                           [&](int i, const Frag<NP> &f) {
                               y = mma(f, xf[i % 2], i % 2 ? y : f32x16{});
                               if (i % 2) {
#pragma unroll
                                   for (int e = 0; e < 16; ++e) acc[i / 2][e] += y[e];
                               }
                           });
    }
}

// ------------------------------------------------------------------------------------------------- forward
// grid: (batch x key head) major, then the part of the states, then the row tile (4 waves x 32 rows).  Two tile buffers: the
// loads of the next tile are issued at the top, written to the other buffer at the bottom, one barrier per tile (three planes:
// one buffer).  (Times here and below are of kernel traces; among repeated calls the large ones are 3 - 10 % shorter.)
// 1,920 x 3,840 x 32 fp32 of 48 heads: 281 - 288 us = 160 TFLOP/s (960 in bf16), the vector units active 0.60 of the time (exponentials,
// cutting into planes) and the matrix units 0.46.  7,680 x 15,360 x 64 bf16 of 8 heads: 340 - 359 us = 690 TFLOP/s, vector 0.45, matrix 0.29: two
// waves per SIMD wait, a third of their cycles for an instruction to be taken.  1,280 x 2,560 x 128 bf16 of 32 heads: 94 us = 570 TFLOP/s, in
// training (P in two planes) 116; vector 0.26, matrix 0.27: 320 workgroups on 256 CUs, one wave per SIMD.
template <int NP, int DP, int BK, bool WIDE, bool TWO>
__global__ void __launch_bounds__(NT) k_attn_fwd(const AttnArgs a)
{
    typedef typename Elem<NP>::T T;
    constexpr int KS = DP / 16, DT = DP / 32, KT = BK / 32;
    constexpr float kMost = 1024.0f;
    __shared__ __attribute__((aligned(16))) Tile<NP, BK, DP> tile_k[buffers(NP)], tile_v[buffers(NP)];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    stagger();
    int id = xcd_run(blockIdx.x, gridDim.x);
    const int tile = id % a.tiles;
    id /= a.tiles;
    const int part = id % a.splits, bh = id / a.splits, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int r = (tile * 4 + wave) * 32 + col;                   // this lane's row
    const bool live = r < a.R;
    const T *kb = (const T *)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[2];
    const T *vb = (const T *)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[2];
    Walk<BK> w(a, b, part, lane);
    Flight<NP, BK, DP, WIDE> fk, fv;
    typedef typename Stride<WIDE>::T Off;
    Off ok[fk.N], ov[fv.N];                                       // rows within a tile
#pragma unroll
    for (int i = 0; i < fk.N; ++i) {
        ok[i] = fk.row_of(i) * (Off)a.ks[1];
        ov[i] = fk.row_of(i) * (Off)a.vs[1];
    }
    auto fetch = [&] {
        auto valid = [&](int row) { return ((uint32_t)(row & 32 ? w.bits >> 32 : w.bits) >> (row & 31)) & 1; };
        const bool all = w.bits == Walk<BK>::kFull;
        fk.fetch(kb + (int64_t)w.j * a.ks[1], a.D, all, valid, [&](int i, int) { return ok[i]; });
        fv.fetch(vb + (int64_t)w.j * a.vs[1], a.D, all, valid, [&](int i, int) { return ov[i]; });
    };
    if (w.live()) fetch();
    Frag<NP> qf[KS];
    const T *qrow = (const T *)a.q + (live ? row_off(a.qs, b, r, hk, a.G) : 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = load8(qrow, 16 * s + 8 * h, a.D, WIDE, live).frag_scaled(a.c);
    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    // reference and sum of the exponentials; sub: the reference, 0 while there is none.  The reference is the maximum of the
    // first tile, and is looked at again only when a sum of exponentials outgrows it (kMost: far from the range of fp32, and
    // bf16 keeps its relative precision): a maximum over every tile would be a sixth of the vector instructions.
    float m = -INFINITY, sub = 0.0f, l = 0.0f;
    constexpr bool kTwo = buffers(NP) == 2;
    bool first = true;
    int buf = 0;
    auto commit = [&] {
        fk.commit(tile_k[buf]);
        fv.commit(tile_v[buf]);
    };
    if (kTwo && w.live()) commit();
    while (w.live()) {
        const uint64_t bits = w.bits;
        const Tile<NP, BK, DP> &tk = tile_k[buf], &tv = tile_v[buf];
        __syncthreads();
        if (!kTwo) {
            commit();
            __syncthreads();
        }
        w.next(a);
        if (w.live()) fetch();
        f32x16 s[KT];
        auto scores = [&] {
#pragma unroll
            for (int t = 0; t < KT; ++t) s[t] = f32x16{};
            stream<NP, KT * KS>([&](int i) { return tk.rows(32 * (i % KT), 16 * (i / KT), lane); },
                                [&](int i, const Frag<NP> &f) { s[i % KT] = mma(f, qf[i / KT], s[i % KT]); });
            if (bits != Walk<BK>::kFull) {
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const uint32_t in = (uint32_t)(bits >> (32 * t)) >> (4 * h);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!((in >> acc_row(i, 0)) & 1)) s[t][i] = -INFINITY;
                }
            }
        };
        auto exps = [&] {
            float lt = 0.0f;
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[t][i] = __builtin_amdgcn_exp2f(exponent<NP>(s[t][i], a.c, -sub));
                    lt += s[t][i];
                }
            return lt;
        };
        scores();
        float lt = 0.0f;
        bool again = first;
        if (!first) {
            lt = exps();
            again = __any(lt > kMost || m == -INFINITY);
            if (again) scores();
        }
        if (again) {
            float mx = s[0][0];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
            mx = fmaxf(other_half_max(mx) * (NP == 3 ? 1.0f : a.c), m);
            sub = mx == -INFINITY ? 0.0f : mx;
            const float f = __builtin_amdgcn_exp2f(m - sub);
            m = mx;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            lt = exps();
        }
        first = false;
        l += lt;
#pragma unroll
        for (int t = 0; t < KT; ++t) accumulate<NP, TWO, true>(o, tv, 32 * t, s[t], lane);
        if (kTwo) {
            buf ^= 1;
            if (w.live()) commit();
        }
    }
    l = other_half_sum(l);
    if (!live) return;
    if (a.splits > 1) {                                          // this part's reference, sum and unscaled output
        const int64_t y = ((int64_t)part * a.B * a.Hk + bh) * a.R + r;
        store_cols<DT>(a.part + y * a.D, o, 1.0f, a.D, (a.D & 3) == 0, h);
        if (h == 0) {
            a.part2[2 * y] = m;
            a.part2[2 * y + 1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store_cols<DT>((T *)a.out + dense_row(b, r, hk, a), o, inv, a.D, (a.D & 3) == 0, h);
    if (TWO && a.low) store_cols_rest<DT>((T *)a.low + dense_row(b, r, hk, a), o, inv, a.D, h);
    if (a.lse && h == 0) store_softmax<NP == 3>(a, (int64_t)bh * a.R + r, m, l);
}

// The same for at most 32 rows (a few queries, or one with the heads of its group): four row tiles would leave three waves of a
// workgroup idle, so here the waves share the rows and divide the states, 32 each in turn, every wave on its own: keys go from
// memory straight to the registers that hold the left operand (32 bytes of a row per lane), values through a tile of the
// wave's own, the next 32 states are in flight meanwhile, and no barrier until the partial results are joined in LDS.
// ROWS: the rows of a product.  At most 16 rows take 16 x 16 x 32 products, half of the matrix work and of the registers of q and o -- but not
// in the forward of an fp32 training step, whose backward has to form the same bits of the scores.
// Bound by the bytes of keys and values: 3.8 TB/s at 15,360 bf16 states (4 x 2 heads of 64: 8.2 us), 3.9 at 40,001 fp32 states (2 x
// 3 heads of 80: 35 us; 43 with 32-row products, 92 by row tiles).
// Eight waves where the registers of 16-row products let two waves into a SIMD and the loads are fp32 (5 x 40,001 x 80: 41.6 us, 43.0
// with four); bf16 keeps four (1 x 15,360 x 64, 4 x 2 heads: 14.1 us, 14.5 with eight, 17 with sixteen).
constexpr int few_waves_of(int NP, int DP, int ROWS) { return NP == 3 && ROWS == 16 && DP <= 96 ? 8 : 4; }
template <int ROWS>
struct AccOf;
template <>
struct AccOf<32> {
    typedef f32x16 T;
};
template <>
struct AccOf<16> {
    typedef f32x4 T;
};
template <int NP, int DP, int ROWS, bool WIDE, bool TWO>
__global__ void __launch_bounds__(64 * few_waves_of(NP, DP, ROWS)) k_attn_few(const AttnArgs a)
{
    typedef typename Elem<NP>::T T;
    typedef typename AccOf<ROWS>::T Acc;
    typedef Tile<NP, 32, DP> VT;
    constexpr int NW = few_waves_of(NP, DP, ROWS), STEP = 32 * NW;              // states of a turn of the workgroup
    constexpr int HN = 64 / ROWS, NE = ROWS * ROWS / 64, KC = 8 * HN;        // lanes of a row, elements of an accumulator, channels of a product
    constexpr int KS = DP / KC, ST = 32 / ROWS, CT = DP / ROWS, LO = DP + 4, NV = 32 * (DP / 8) / 64;
    constexpr size_t kTiles = NW * sizeof(VT), kOut = NW * ROWS * LO * sizeof(float);
    __shared__ __attribute__((aligned(16))) char mem[kTiles > kOut ? kTiles : kOut];
    __shared__ float wave_m[NW][ROWS], wave_l[NW][ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & (ROWS - 1), h = lane / ROWS;
    const int id = xcd_run(blockIdx.x, gridDim.x), part = id % a.splits, bh = id / a.splits, b = bh / a.Hk, hk = bh - b * a.Hk;
    VT &tv = ((VT *)mem)[wave];
    const T *kb = (const T *)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[2];
    const T *vb = (const T *)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[2];
    const typename Stride<WIDE>::T ks = a.ks[1], vs = a.vs[1];
    const int n = states_of(a, b), end = (int)min((int64_t)n, (int64_t)(part + 1) * a.per * STEP);
    int j = part * a.per * STEP + wave * 32;
    uint32_t bits = 0;
    auto settle = [&] {                                           // on to 32 states of which one counts
        for (; j < end; j += STEP) {
            bits = (uint32_t)live_states(a, b, j, n, lane);
            if (bits) return;
        }
    };
    Raw<NP> rk[ST * KS], rv[NV];
    auto fetch = [&] {
        const T *kt = kb + (int64_t)j * a.ks[1], *vt = vb + (int64_t)j * a.vs[1];
        if constexpr (WIDE) {
            const __amdgpu_buffer_rsrc_t sk = __builtin_amdgcn_make_buffer_rsrc((void *)uniform_ptr(kt), (short)0, 0x7fffffff, 0x00027000);
            const __amdgpu_buffer_rsrc_t sv = __builtin_amdgcn_make_buffer_rsrc((void *)uniform_ptr(vt), (short)0, 0x7fffffff, 0x00027000);
#pragma unroll
            for (int x = 0; x < ST * KS; ++x) {
                const int row = x / KS * ROWS + col, d = KC * (x % KS) + 8 * h;
                rk[x].load(sk, ((bits >> row) & 1) && d < a.D ? (uint32_t)(row * ks + d) * (uint32_t)sizeof(T) : kNowhere, d + 4 < a.D);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = i * 64 + lane, row = c / (DP / 8), d = (c - row * (DP / 8)) * 8;
                rv[i].load(sv, ((bits >> row) & 1) && d < a.D ? (uint32_t)(row * vs + d) * (uint32_t)sizeof(T) : kNowhere, d + 4 < a.D);
            }
        } else {
#pragma unroll
            for (int x = 0; x < ST * KS; ++x) {
                const int row = x / KS * ROWS + col;
                const bool in = (bits >> row) & 1;
                rk[x] = load8(kt + (in ? row * ks : 0), KC * (x % KS) + 8 * h, a.D, false, in);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = i * 64 + lane, row = c / (DP / 8), d = (c - row * (DP / 8)) * 8;
                const bool in = (bits >> row) & 1;
                rv[i] = load8(vt + (in ? row * vs : 0), d, a.D, false, in);
            }
        }
    };
    settle();
    if (j < end) fetch();
    const bool live = col < a.R;
    const T *qrow = (const T *)a.q + (live ? row_off(a.qs, b, col, hk, a.G) : 0);
    Frag<NP> qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = load8(qrow, KC * s + 8 * h, a.D, WIDE, live).frag_scaled(a.c);
    Acc o[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) o[t] = Acc{};
    auto across_max = [](float x) { return other_half_max(ROWS == 16 ? other_row_max(x) : x); };
    auto state = [&](int t, int i) { return ROWS == 32 ? acc_row(i, 0) : 16 * t + i; };       // of element i of tile t, before 4 h
    float m = -INFINITY, l = 0.0f;
    while (j < end) {
        const uint32_t ok = bits >> (4 * h);
        Acc s[ST];
#pragma unroll
        for (int t = 0; t < ST; ++t) {
            s[t] = Acc{};
#pragma unroll
            for (int x = 0; x < KS; ++x) s[t] = mma(rk[t * KS + x].frag(), qf[x], s[t]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = i * 64 + lane, row = c / (DP / 8);
            tv.put(row, c - row * (DP / 8), rv[i].frag());
        }
        __builtin_amdgcn_wave_barrier();                          // (LDS accesses of one wave are in order)
        j += STEP;
        settle();
        if (j < end) fetch();
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                if (!((ok >> state(t, i)) & 1)) s[t][i] = -INFINITY;
                mx = fmaxf(mx, s[t][i]);
            }
        mx = fmaxf(across_max(mx) * (NP == 3 ? 1.0f : a.c), m);
        const float sub = mx == -INFINITY ? 0.0f : mx, f = __builtin_amdgcn_exp2f(m - sub);
        m = mx;
        float lt = 0.0f;
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(exponent<NP>(s[t][i], a.c, -sub));
                lt += s[t][i];
            }
        l = fmaf(l, f, lt);
#pragma unroll
        for (int d = 0; d < CT; ++d)
#pragma unroll
            for (int i = 0; i < NE; ++i) o[d][i] *= f;
        if constexpr (ROWS == 32) {
            accumulate<NP, TWO, true>(o, tv, 0, s[0], lane);
        } else {
            const float p[8] = {s[0][0], s[0][1], s[0][2], s[0][3], s[1][0], s[1][1], s[1][2], s[1][3]};
            Frag<NP> pf, low;
            if constexpr (TWO) split8<true>(p, pf, low);
            else pf = split8<NP>(p);
            stream<NP, CT>([&](int i) { return tv.cols16(16 * i, lane); },
                           [&](int i, const Frag<NP> &vf) {
                               if constexpr (TWO) {
                                   o[i] = mma(vf, pf, mma(vf, low, o[i]));
                               } else if constexpr (NP == 1) {
                                   o[i] = mma(vf, pf, o[i]);
                               } else {
                                   const f32x4 y = mma(vf, pf, f32x4{});      // (summed on its own, as in accumulate)
#pragma unroll
                                   for (int e = 0; e < 4; ++e) o[i][e] += y[e];
                               }
                           });
        }
        __builtin_amdgcn_wave_barrier();
    }
    l = other_half_sum(ROWS == 16 ? other_row_sum(l) : l);
    __syncthreads();                                              // the value tiles are read: their memory takes the partial outputs
    float *out = (float *)mem;
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int i = 0; i < NE / 4; ++i)
            *(f32x4 *)&out[(wave * ROWS + col) * LO + ROWS * t + 8 * i + 4 * h] = f32x4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
    if (h == 0) {
        wave_m[wave][col] = m;
        wave_l[wave][col] = l;
    }
    __syncthreads();
    constexpr int LPR = 64 * NW / ROWS;                           // lanes per row
    const int r = threadIdx.x / LPR, c = threadIdx.x % LPR;
    if (r >= a.R) return;
    float f[NW], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w)
        if (wave_l[w][r] != 0.0f) top = fmaxf(top, wave_m[w][r]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        f[w] = wave_l[w][r] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(wave_m[w][r] - top);
        sum = fmaf(wave_l[w][r], f[w], sum);
    }
    const int64_t y = ((int64_t)part * a.B * a.Hk + bh) * a.R + r;
    const float inv = a.splits > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int d = 4 * c; d < DP; d += 4 * LPR) {
        f32x4 x = {};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (f[w] != 0.0f) x[i] = fmaf(out[(w * ROWS + r) * LO + d + i], f[w], x[i]);
        if (a.splits > 1) store4(a.part + y * a.D, d, a.D, (a.D & 3) == 0, x[0], x[1], x[2], x[3]);
        else {
            store4((T *)a.out + dense_row(b, r, hk, a), d, a.D, (a.D & 3) == 0, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            if (TWO && a.low) store_rest((T *)a.low + dense_row(b, r, hk, a), d, a.D, {x[0], x[1], x[2], x[3]}, inv);
        }
    }
    if (c == 0) {
        if (a.splits > 1) {
            a.part2[2 * y] = top;
            a.part2[2 * y + 1] = sum;
        } else if (a.lse) {
            store_softmax<NP == 3>(a, (int64_t)bh * a.R + r, top, sum);
        }
    }
}

// ------------------------------------------------------------------------------------------------- backward
// P is recomputed from the reference and the sum of the row's exponentials (store_softmax); delta = do . o is what the softmax subtracts from dP:
//     dS = P (dP - delta),  dP = do V^T,  dq = scale dS K,  dk = scale dS^T q,  dv = P^T do
// (delta is summed in fp32 from do and the output.  In bf16 the forward of a training step forms the output from two planes of P and stores what
// its rounding left as well: the rounded output alone makes dS that do not sum to zero, and dq and dk up to 1.9 times as far off as
// their own rounding, 4.8 times with dS in one plane as well, where few states share the weight.  It costs 5 % of a training call, 427 -> 449
// us at 4 x 1,280 x 2,560 x 128; dS in two planes for dq another 16 us.)
// Two passes without atomics, so that the sums have one order: rows own dq (and write delta), states own dk and dv.  The
// heads that share keys are rows of the same loop, so their gradients add up in the accumulator.

// dP - delta: the products of dP start from -delta where sixteen registers more do not cost a wave per SIMD (1,280 x 2,560 x 128
// bf16 backward: 311 -> 343 us).  (The scores do not start from -lse: it outweighs their terms, and each sum would round at its
// size -- dk and dv of 120 x 240 x 64 fp32: 4e-7 -> 1e-6 of the result.)
constexpr bool start_at_delta(int NP, int DP) { return NP == 3 || DP <= 64; }

// grid as the forward's: S^T and dP^T of a tile, then dq^T += K^T dS^T.  1,920 x 3,840 x 32 fp32 of 48 heads: 367 - 375 us = 183 TFLOP/s, matrix
// units 0.55, vector units 0.50 of the time; 1,280 x 2,560 x 128 bf16 of 32 heads: 143 us (119 with dS in one plane), 0.30 and 0.24.
template <int NP, int DP, int BK, bool WIDE>
__global__ void __launch_bounds__(NT) k_attn_dq(const AttnArgs a)
{
    typedef typename Elem<NP>::T T;
    constexpr int KS = DP / 16, DT = DP / 32, KT = BK / 32;
    __shared__ __attribute__((aligned(16))) Tile<NP, BK, DP> tile_k[buffers(NP)], tile_v[buffers(NP)];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    stagger();
    int id = xcd_run(blockIdx.x, gridDim.x);
    const int tile = id % a.tiles;
    id /= a.tiles;
    const int part = id % a.splits, bh = id / a.splits, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int r = (tile * 4 + wave) * 32 + col;
    const bool live = r < a.R, dwide = WIDE || a.D % (16 / (int)sizeof(T)) == 0;      // whole 16-byte runs in the dense rows
    const T *kb = (const T *)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[2];
    const T *vb = (const T *)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[2];
    Walk<BK> w(a, b, part, lane);
    Flight<NP, BK, DP, WIDE> fk, fv;
    typedef typename Stride<WIDE>::T Off;
    Off ok[fk.N], ov[fv.N];                                       // rows within a tile
#pragma unroll
    for (int i = 0; i < fk.N; ++i) {
        ok[i] = fk.row_of(i) * (Off)a.ks[1];
        ov[i] = fk.row_of(i) * (Off)a.vs[1];
    }
    auto fetch = [&] {
        auto valid = [&](int row) { return ((uint32_t)(row & 32 ? w.bits >> 32 : w.bits) >> (row & 31)) & 1; };
        const bool all = w.bits == Walk<BK>::kFull;
        fk.fetch(kb + (int64_t)w.j * a.ks[1], a.D, all, valid, [&](int i, int) { return ok[i]; });
        fv.fetch(vb + (int64_t)w.j * a.vs[1], a.D, all, valid, [&](int i, int) { return ov[i]; });
    };
    if (w.live()) fetch();
    Frag<NP> qf[KS], gf[KS];
    const T *qrow = (const T *)a.q + (live ? row_off(a.qs, b, r, hk, a.G) : 0);
    const int64_t dense = live ? dense_row(b, r, hk, a) : 0;
    float delta = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        qf[s] = load8(qrow, 16 * s + 8 * h, a.D, WIDE, live).frag_scaled(a.c);
        const Raw<NP> g = load8((const T *)a.go + dense, 16 * s + 8 * h, a.D, dwide, live);
        delta = dot8(g, load8((const T *)a.o + dense, 16 * s + 8 * h, a.D, dwide, live), delta);
        if (NP == 1 && a.low) delta = dot8(g, load8((const T *)a.low + dense, 16 * s + 8 * h, a.D, dwide, live), delta);
        gf[s] = g.frag();
    }
    delta = other_half_sum(delta);
    const float lse = live ? a.lse[(int64_t)bh * a.R + r] : INFINITY;
    const float out = NP == 3 && a.inv && live ? a.scale * a.inv[(int64_t)bh * a.R + r] : a.scale;      // of the sums below, the row's dq
    if (live && part == 0 && h == 0) a.delta[(int64_t)bh * a.R + r] = delta;
    f32x16 dq[DT], minus_delta;
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = f32x16{};
#pragma unroll
    for (int i = 0; i < 16; ++i) minus_delta[i] = -delta;
    constexpr bool kTwo = buffers(NP) == 2;
    int buf = 0;
    auto commit = [&] {
        fk.commit(tile_k[buf]);
        fv.commit(tile_v[buf]);
    };
    if (kTwo && w.live()) commit();
    while (w.live()) {
        const uint64_t bits = w.bits;
        const Tile<NP, BK, DP> &tk = tile_k[buf], &tv = tile_v[buf];
        __syncthreads();
        if (!kTwo) {
            commit();
            __syncthreads();
        }
        w.next(a);
        if (w.live()) fetch();
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            f32x16 s = {}, dp = {};
            if (start_at_delta(NP, DP)) dp = minus_delta;
            stream<NP, 2 * KS>([&](int i) { return (i % 2 ? tv : tk).rows(32 * t, 16 * (i / 2), lane); },
                               [&](int i, const Frag<NP> &f) {
                                   if (i % 2) dp = mma(f, gf[i / 2], dp);
                                   else s = mma(f, qf[i / 2], s);
                               });
            // a state that does not count: its row of the tile is zero, so whatever dS holds for it adds nothing to dq --
            // but exp2(-lse) may be infinite there, so it is cleared
            if (bits != Walk<BK>::kFull) {
                const uint32_t in = (uint32_t)(bits >> (32 * t)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!((in >> acc_row(i, 0)) & 1)) s[i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = __builtin_amdgcn_exp2f(exponent<NP>(s[i], a.c, -lse)) * (start_at_delta(NP, DP) ? dp[i] : dp[i] - delta);
            accumulate<NP, NP == 1, false>(dq, tk, 32 * t, s, lane);
        }
        if (kTwo) {
            buf ^= 1;
            if (w.live()) commit();
        }
    }
    if (!live) return;
    if (a.splits > 1) {
        const int64_t y = ((int64_t)part * a.B * a.Hk + bh) * a.R + r;
        store_cols<DT>(a.part + y * a.D, dq, out, a.D, (a.D & 3) == 0, h);
        return;
    }
    store_cols<DT>((T *)a.dq + dense, dq, out, a.D, (a.D & 3) == 0, h);
}

// grid: (batch x key head) major, then the part of the rows, then the state tile (4 waves x 32 states).  Row tiles of q and do
// are staged; S and dP have this wave's states as columns, dv^T += do^T P, dk^T += q^T dS.  1,920 x 3,840 x 32 fp32 of 48 heads:
// 522 us = 174 TFLOP/s, matrix units 0.51, vector units 0.53 of the time; 1,280 x 2,560 x 128 bf16 of 32 heads: 217 us = 490 TFLOP/s, 0.19 and
// 0.17: dk, dv, k and v in registers leave one wave per SIMD.
template <int NP, int DP, int BQ, bool WIDE, bool TWO>
__global__ void __launch_bounds__(NT) k_attn_dkv(const AttnArgs a)
{
    typedef typename Elem<NP>::T T;
    constexpr int KS = DP / 16, DT = DP / 32, QT = BQ / 32;
    __shared__ __attribute__((aligned(16))) Tile<NP, BQ, DP> tile_q[buffers(NP)], tile_g[buffers(NP)];
    __shared__ __attribute__((aligned(16))) float row_lse[buffers(NP)][BQ], row_delta[buffers(NP)][BQ];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    stagger();
    int id = xcd_run(blockIdx.x, gridDim.x);
    const int tile = id % a.tiles;
    id /= a.tiles;
    const int part = id % a.splits, bh = id / a.splits, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int j = (tile * 4 + wave) * 32 + col, n = states_of(a, b);
    const int r1 = tile * 128 < n ? (int)min((int64_t)a.R, (int64_t)(part + 1) * a.per * BQ) : 0;
    int r0 = part * a.per * BQ;
    Flight<NP, BQ, DP, WIDE> fq, fg;
    float pl = 0.0f, pd = 0.0f, pf[fg.N];                        // pf: what do and delta of a row are multiplied with, in place of P
    typedef typename Stride<WIDE>::T Off;
    const Off qs1 = a.qs[1], qs2 = a.qs[2], gs1 = (int64_t)a.Hq * a.D, gs2 = a.D;
    const float invG = 1.0f / (float)a.G;
    auto fetch = [&] {
        // row r0 + row is token i0 + i, head g of the group: (g0 + row) / G by a product, exact for the small numbers that come up
        // (G <= kMaxGroup; half a unit away from every integer)
        const int i0 = r0 / a.G, g0 = r0 - i0 * a.G;
        auto valid = [&](int row) { return r0 + row < a.R; };
        auto token = [&](int row) { return (int)(((float)(g0 + row) + 0.5f) * invG); };
        const T *qb = (const T *)a.q + (int64_t)b * a.qs[0] + (int64_t)hk * a.G * a.qs[2] + (int64_t)i0 * a.qs[1];
        const T *gb = (const T *)a.go + (((int64_t)b * a.Lq + i0) * a.Hq + (int64_t)hk * a.G) * a.D;
        const bool all = r0 + BQ <= a.R;
        fq.fetch(qb, a.D, all, valid, [&](int, int row) { const int i = token(row); return i * qs1 + (g0 + row - i * a.G) * qs2; });
        fg.fetch(gb, a.D, all, valid, [&](int, int row) { const int i = token(row); return i * gs1 + (g0 + row - i * a.G) * gs2; });
        if (threadIdx.x < BQ) {
            const int r = r0 + threadIdx.x;
            pl = r < a.R ? -a.lse[(int64_t)bh * a.R + r] : -INFINITY;          // rows behind the last: P = 0
            pd = r < a.R ? -a.delta[(int64_t)bh * a.R + r] : 0.0f;
            if (NP == 3 && a.inv && r < a.R) pd *= a.inv[(int64_t)bh * a.R + r];
        }
        if constexpr (NP == 3) {
#pragma unroll
            for (int i = 0; i < fg.N; ++i) {
                const int r = r0 + fg.row_of(i);
                pf[i] = a.inv && r < a.R ? a.inv[(int64_t)bh * a.R + r] : 1.0f;
            }
        }
    };
    constexpr bool kTwo = buffers(NP) == 2;
    int buf = 0;
    auto commit = [&] {
        if constexpr (NP == 3) {
            fq.commit(tile_q[buf], [&](int) { return a.c; });
            fg.commit(tile_g[buf], [&](int i) { return pf[i]; });
        } else {
            fq.commit(tile_q[buf]);
            fg.commit(tile_g[buf]);
        }
        if (threadIdx.x < BQ) {
            row_lse[buf][threadIdx.x] = pl;
            row_delta[buf][threadIdx.x] = pd;
        }
    };
    if (r0 < r1) fetch();
    const bool live = j < n && (!a.mask || a.mask[(int64_t)b * a.ms[0] + (int64_t)j * a.ms[1]] != 0);
    const T *krow = (const T *)a.k + (live ? (int64_t)b * a.ks[0] + (int64_t)j * a.ks[1] + (int64_t)hk * a.ks[2] : 0);
    const T *vrow = (const T *)a.v + (live ? (int64_t)b * a.vs[0] + (int64_t)j * a.vs[1] + (int64_t)hk * a.vs[2] : 0);
    Frag<NP> kf[KS], vf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        kf[s] = load_frag<NP>(krow, 16 * s + 8 * h, a.D, WIDE, live);
        vf[s] = load_frag<NP>(vrow, 16 * s + 8 * h, a.D, WIDE, live);
    }
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) dk[d] = dv[d] = f32x16{};
    if (kTwo && r0 < r1) commit();
    while (r0 < r1) {
        const Tile<NP, BQ, DP> &tq = tile_q[buf], &tg = tile_g[buf];
        const float *sl = row_lse[buf], *sd = row_delta[buf];
        __syncthreads();
        if (!kTwo) {
            commit();
            __syncthreads();
        }
        r0 += BQ;
        if (r0 < r1) fetch();
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            constexpr bool kStart = start_at_delta(NP, DP);
            f32x16 s = {}, dp = {};
            auto row4 = [&](const float *x, int i) { return *(const f32x4 *)&x[32 * u + acc_row(4 * i, h)]; };     // of elements 4 i ..
            if (kStart) {
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] = row4(sd, i / 4)[i % 4];
            }
            stream<NP, 2 * KS>([&](int i) { return (i % 2 ? tg : tq).rows(32 * u, 16 * (i / 2), lane); },
                               [&](int i, const Frag<NP> &f) {
                                   if (i % 2) dp = mma(f, vf[i / 2], dp);
                                   else s = mma_exchanged(f, kf[i / 2], s);
                               });
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                // (the column of a state that does not count is dropped at the end)
                s[i] = __builtin_amdgcn_exp2f(exponent<NP>(s[i], a.c, row4(sl, i / 4)[i % 4]));
                dp[i] = s[i] * (kStart ? dp[i] : dp[i] + row4(sd, i / 4)[i % 4]);
            }
            accumulate<NP, TWO, true>(dv, tg, 32 * u, s, lane);
            accumulate<NP, TWO, false>(dk, tq, 32 * u, dp, lane);
        }
        if (kTwo) {
            buf ^= 1;
            if (r0 < r1) commit();
        }
    }
    if (j >= a.Lk) return;
    const float of_dk = NP == 3 ? kLn2 : a.scale;                 // (three planes: the rows carry scale * log2(e))
    if (!live) {
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[d] = dv[d] = f32x16{};
    }
    if (a.splits > 1) {
        const int64_t n1 = (int64_t)a.B * a.Hk * a.Lk * a.D, y = ((int64_t)bh * a.Lk + j) * a.D + 2 * part * n1;
        const bool pw = (a.D & 3) == 0;
        store_cols<DT>(a.part + y, dk, of_dk, a.D, pw, h);
        store_cols<DT>(a.part + y + n1, dv, 1.0f, a.D, pw, h);
        return;
    }
    const int64_t y = (((int64_t)b * a.Lk + j) * a.Hk + hk) * a.D;
    store_cols<DT>((T *)a.dk + y, dk, of_dk, a.D, (a.D & 3) == 0, h);
    store_cols<DT>((T *)a.dv + y, dv, 1.0f, a.D, (a.D & 3) == 0, h);
}

// ------------------------------------------------------------------------------------------------- joining parts
// `wpr` waves per row (four where rows are few, else one): `per` lanes hold four channels each, the groups of lanes of all its
// waves take the parts in turn, a butterfly adds the groups of a wave and LDS the waves: one fixed order.  (A lane that walked
// 60 parts by itself took 56 us of a single-token call, a wave per row 11 us of 42 parts of 80 channels.)
//   MODE 0: o = sum_p o_p 2^(m_p - m) / sum_p l_p 2^(m_p - m), and the row's lse
//   MODE 1: dq = sum_p dq_p;  MODE 2: dk and dv, part[p][2][B * Hk][Lk][D]
template <typename T, int MODE>
__global__ void __launch_bounds__(NT) k_attn_join(const AttnArgs a, int per, int wpr, int64_t total)
{
    __shared__ f32x4 wave_o[3][32];
    const int wave = threadIdx.x >> 6, sub = wave & (wpr - 1), lane = threadIdx.x & 63, c = lane & (per - 1), pg = lane / per, groups = 64 / per, d = 4 * c;
    const int64_t row = (int64_t)blockIdx.x * (NT / 64 / wpr) + wave / wpr;
    if (row >= total) return;                                    // (the waves of a row together)
    const int len = MODE == 2 ? a.Lk : a.R;
    const int64_t rows = (int64_t)a.B * a.Hk * len;
    const int which = MODE == 2 && row >= rows;
    const int64_t w = which ? row - rows : row;
    float f = 1.0f, l = 0.0f, m = 0.0f;
    if (MODE == 0) {                                             // (at most 64 parts: one per lane)
        const bool in = lane < a.splits;
        const float lp = in ? a.part2[2 * (lane * rows + w) + 1] : 0.0f, mp = in && lp != 0.0f ? a.part2[2 * (lane * rows + w)] : -INFINITY;
        m = mp;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
        f = lp == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mp - m);  // parts without a state that counts: weight 0
        l = lp * f;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x, 64);
    }
    float o[4] = {0, 0, 0, 0};
    const bool quad = (a.D & 3) == 0;
    const int64_t step = (MODE == 2 ? 2 : 1) * rows * a.D;
    const float *src = a.part + (which * rows + w) * a.D + d;
#pragma unroll 8
    for (int p0 = sub * groups; p0 < a.splits; p0 += groups * wpr) {
        const int p = p0 + pg;
        const float wt = MODE == 0 ? __shfl(f, p & 63, 64) : 1.0f;
        if (p < a.splits && d < a.D && wt != 0.0f) {
            const float *y = src + p * step;
            if (quad) {
                const f32x4 v = *(const f32x4 *)y;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = fmaf(v[i], wt, o[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < a.D) o[i] = fmaf(y[i], wt, o[i]);
            }
        }
    }
    for (int x = per; x < 64; x <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x, 64);
    if (wpr > 1) {                                               // (per <= 32: one row per workgroup)
        if (sub && !pg) wave_o[sub - 1][c] = f32x4{o[0], o[1], o[2], o[3]};
        __syncthreads();
        if (sub) return;
#pragma unroll
        for (int w1 = 0; w1 < 3; ++w1)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += wave_o[w1][c][i];
    }
    if (pg) return;
    const int bh = (int)(w / len), r = (int)(w - (int64_t)bh * len), b = bh / a.Hk, hk = bh - b * a.Hk;
    const float inv = MODE == 0 ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
    T *dst = MODE == 2 ? (T *)(which ? a.dv : a.dk) + (((int64_t)b * a.Lk + r) * a.Hk + hk) * a.D
                       : (T *)(MODE == 0 ? a.out : a.dq) + dense_row(b, r, hk, a);
    store4(dst, d, a.D, (a.D & 3) == 0, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (MODE == 0 && a.low) store_rest((T *)a.low + dense_row(b, r, hk, a), d, a.D, o, inv);
    if (MODE == 0 && a.lse && c == 0) store_softmax<sizeof(T) == 4>(a, w, m, l);
}

// The same for few parts (at most kFlat): a lane adds all parts of its four channels, without a word to the others.  (Two parts of
// 120 x 240 x 64 fp32, 96 heads: 24.0 -> 20.3 us forward, 48.2 -> 46.3 backward by events around the launches -- an eager training call
// is the host's, 71 - 74 us either way; eight parts alike in both forms, sixteen 2 us slower.)
constexpr int kFlat = 4;
template <typename T, int MODE>
__global__ void __launch_bounds__(NT) k_attn_join_flat(const AttnArgs a, int per, int64_t total)
{
    const int d = 4 * (threadIdx.x & (per - 1));
    const int64_t row = (int64_t)blockIdx.x * (NT / per) + threadIdx.x / per;
    if (row >= total || d >= a.D) return;
    const int len = MODE == 2 ? a.Lk : a.R;
    const int64_t rows = (int64_t)a.B * a.Hk * len;
    const int which = MODE == 2 && row >= rows;
    const int64_t w = which ? row - rows : row;
    float f[kFlat], m = -INFINITY, l = 0.0f;
    if (MODE == 0) {
        float mp[kFlat];
#pragma unroll
        for (int p = 0; p < kFlat; ++p) {
            const float *y = a.part2 + 2 * (min(p, a.splits - 1) * rows + w);
            mp[p] = y[0];
            f[p] = p < a.splits ? y[1] : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < kFlat; ++p)
            if (f[p] != 0.0f) m = fmaxf(m, mp[p]);
#pragma unroll
        for (int p = 0; p < kFlat; ++p) {
            const float lp = f[p];
            f[p] = lp == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mp[p] - m);      // parts without a state that counts: weight 0
            l = fmaf(lp, f[p], l);
        }
    }
    float o[4] = {0, 0, 0, 0};
    const bool quad = (a.D & 3) == 0;
    const int64_t step = (MODE == 2 ? 2 : 1) * rows * a.D;
    const float *src = a.part + (which * rows + w) * a.D + d;
#pragma unroll
    for (int p = 0; p < kFlat; ++p) {
        const float wt = MODE == 0 ? f[p] : 1.0f;
        if (p < a.splits && wt != 0.0f) {
            const float *y = src + p * step;
            if (quad) {
                const f32x4 v = *(const f32x4 *)y;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = fmaf(v[i], wt, o[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < a.D) o[i] = fmaf(y[i], wt, o[i]);
            }
        }
    }
    const int bh = (int)(w / len), r = (int)(w - (int64_t)bh * len), b = bh / a.Hk, hk = bh - b * a.Hk;
    const float inv = MODE == 0 ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
    T *dst = MODE == 2 ? (T *)(which ? a.dv : a.dk) + (((int64_t)b * a.Lk + r) * a.Hk + hk) * a.D
                       : (T *)(MODE == 0 ? a.out : a.dq) + dense_row(b, r, hk, a);
    store4(dst, d, a.D, quad, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (MODE == 0 && a.low) store_rest((T *)a.low + dense_row(b, r, hk, a), d, a.D, o, inv);
    if (MODE == 0 && a.lse && d == 0) store_softmax<sizeof(T) == 4>(a, w, m, l);
}

// ------------------------------------------------------------------------------------------------- host side

// parts of a reduction of `red` tiles when `blocks` workgroups exist without splitting: as many as fit one workgroup per CU,
// with at least `least` tiles each, at most 64.  (More cost more in the parts' round trip through memory than the evener load
// gives, in calls: 480 workgroups, 7,680 x 15,360 x 64 bf16: 321 us in one part, 338 in two; 16 of 480 x 9,600 x 64 bf16: 22 us in 16 parts, 27
// in 32; 72 of 333 x 1,281 x 28 fp32: 34 us in two, 27 in three; 6 of 5 x 40,001 x 80 fp32: 41.5 us in 40, 56 in 64.  The exception,
// 192 of 480 x 960 x 32 backward: 67 us in one, 64 in two.)
constexpr int kCUs = 256;
void split_of(int64_t blocks, int red, int least, int &splits, int &per)
{
    int64_t s = blocks > 0 ? kCUs / blocks : 1;
    if (s > 64) s = 64;
    if (s > red / least) s = red / least;
    if (s < 1) s = 1;
    per = (int)((red + s - 1) / s);
    if (per < 1) per = 1;
    splits = red > 0 ? (red + per - 1) / per : 1;
}

// states of a staged tile
constexpr int tile_states(int NP, int DP) { return NP == 1 || DP <= 32 ? 64 : 32; }
// rows of a staged tile of the dk / dv kernel
constexpr int tile_rows(int NP, int DP) { return DP <= (NP == 1 ? 64 : 32) ? 64 : 32; }
constexpr int kMaxGroup = 65536;                                 // query heads of a head of states (k_attn_dkv divides by a product)

// whether 16-byte loads fit: aligned rows, and 32-bit byte offsets within a tile of 64 rows or states
bool wide_rows(const mvf_attn_desc &d)
{
    const int64_t align = d.dtype == MVF_DTYPE_BF16 ? 8 : 4, G = d.Hq / d.Hk, most = 0x7fffffffLL / 4 - 128;
    if (d.D % align) return false;
    for (int i = 0; i < 3; ++i)
        if (d.q_stride[i] % align || d.k_stride[i] % align || d.v_stride[i] % align) return false;
    if (((uintptr_t)d.q | (uintptr_t)d.k | (uintptr_t)d.v) & 15) return false;
    const int64_t *q = d.q_stride, *k = d.k_stride, *v = d.v_stride;
    if (q[1] < 0 || q[2] < 0 || k[1] < 0 || v[1] < 0 || q[1] > most || q[2] > most || k[1] > most / 64 || v[1] > most / 64) return false;
    // (64 rows reach over 63 / G + 2 tokens, and the G heads of one)
    return (63 / G + 2) * q[1] + G * q[2] <= most && ((63 / G + 2) * d.Hq + G) * d.D <= most;
}

// Two planes of P and dS where one would be as much again as the result's own rounding, or more, and where they cost nothing:
//   * the forward of a training step, whose output and its rest make delta;
//   * dq: the dS of a row sum to zero and the keys that share its weight are alike, so that its terms cancel and their roundings do not
//     (in one plane 1.5 times its own rounding, 2 in all, with normal queries and keys of 6 channels or four times larger queries of 16);
//   * all of them below kSmall operations of the two forward products: an eager call of that size is the host's; in a captured training
//     step they cost 1 - 4 us of 25 - 37 (60 x 120 and 120 x 240 x 64, 96 heads), 9 of 142 at one query and 15,360 states.
// Everywhere they would cost 12 - 27 % (training 12 x 1,920 x 3,840 of 4 x 32: 335 -> 424 us; 4 x 1,280 x 2,560 of 8 x 128: 447 -> 499).
constexpr double kSmall = 1e9;

struct Plan {
    bool wide;                               // 16-byte loads
    int NP, DP, BK, BQ;
    int rtiles, ktiles;                      // workgroups along the rows, along the states
    int few;                                 // forward of at most 32 rows, the waves divide the states: 16 or 32 rows of a product; 0: more
    bool two_f, two_k;                       // bf16: P and dS as two planes in the forward, dk / dv
    int fs, fper, qs, qper, ks, kper;        // parts of the reduction and tiles of a part: forward, dq (over the states), dkv (over the rows)
};
Plan plan_of(const mvf_attn_desc &d)
{
    Plan p;
    p.wide = wide_rows(d);
    p.NP = d.dtype == MVF_DTYPE_F32 ? 3 : 1;
    p.DP = d.D <= 32 ? 32 : d.D <= 64 ? 64 : d.D <= 96 ? 96 : 128;
    p.BK = tile_states(p.NP, p.DP);
    p.BQ = tile_rows(p.NP, p.DP);
    const int R = d.Lq * (d.Hq / d.Hk);
    const int64_t bh = (int64_t)d.B * d.Hk;
    const bool small = 4.0 * bh * R * d.Lk * d.D < kSmall;
    p.two_f = p.NP == 1 && (d.out_low || small);
    p.two_k = p.NP == 1 && small;
    p.rtiles = (R + 127) / 128;
    p.ktiles = (d.Lk + 127) / 128;
    p.few = R <= 16 && !(p.NP == 3 && d.inv_sum) ? 16 : R <= 32 ? 32 : 0;       // (an fp32 backward forms the scores of 32-row products)
    split_of(bh * p.rtiles, (d.Lk + p.BK - 1) / p.BK, 4, p.qs, p.qper);
    const int turn = 32 * few_waves_of(p.NP, p.DP, p.few);
    if (p.few) split_of(bh, (d.Lk + turn - 1) / turn, 256 / turn, p.fs, p.fper);
    else p.fs = p.qs, p.fper = p.qper;
    split_of(bh * p.ktiles, (R + p.BQ - 1) / p.BQ, 4, p.ks, p.kper);
    return p;
}
bool bad_desc(const mvf_attn_desc *d)
{
    if (!d || d->B < 0 || d->Lq < 0 || d->Lk < 0 || d->Hq <= 0 || d->Hk <= 0 || d->Hq % d->Hk || d->D <= 0 || d->D > MVF_ATTN_MAX_D) return true;
    if (d->dtype != MVF_DTYPE_F32 && d->dtype != MVF_DTYPE_BF16) return true;
    if (!(d->scale > 0.0f) || !(d->scale * kLog2e < INFINITY)) return true;
    if (d->Hq / d->Hk > kMaxGroup) return true;
    const int64_t G = d->Hq / d->Hk, R = G * d->Lq, bh = (int64_t)d->B * d->Hk;
    // 32-bit tile counts (offsets into the tensors are 64-bit throughout)
    if (R > (1 << 30) || d->Lk > (1 << 30) || bh > 0x7fffffffLL) return true;
    // and launches that the runtime takes, of the forward and of both kernels of the backward (parts exist only of far fewer workgroups)
    const Plan p = plan_of(*d);
    const int64_t fwd = p.few ? bh * 64 * few_waves_of(p.NP, p.DP, p.few) : bh * p.rtiles * NT;
    return fwd > kMaxThreads || bh * p.rtiles * NT > kMaxThreads || bh * p.ktiles * NT > kMaxThreads;
}
AttnArgs args_of(const mvf_attn_desc &d, const Plan &p)
{
    AttnArgs a = {};
    a.q = d.q; a.k = d.k; a.v = d.v;
    a.low = d.dtype == MVF_DTYPE_BF16 ? d.out_low : nullptr;
    a.inv = d.dtype == MVF_DTYPE_F32 ? d.inv_sum : nullptr;
    a.mask = d.key_mask; a.lens = d.kv_lens;
    for (int i = 0; i < 3; ++i) { a.qs[i] = d.q_stride[i]; a.ks[i] = d.k_stride[i]; a.vs[i] = d.v_stride[i]; }
    a.wide = p.wide;
    a.ms[0] = d.mask_stride[0]; a.ms[1] = d.mask_stride[1];
    a.B = d.B; a.Lq = d.Lq; a.Lk = d.Lk; a.Hq = d.Hq; a.Hk = d.Hk; a.D = d.D;
    a.G = d.Hq / d.Hk;
    a.R = d.Lq * a.G;
    a.scale = d.scale;
    a.c = d.scale * kLog2e;
    return a;
}

// a kernel by its last two arguments, 16-byte loads and two planes (of one-plane inputs alone)
#define MVF_ATTN_LAUNCH(two, g, b, st, a, ...)                                                         \
    do {                                                                                               \
        if constexpr (NP == 1) {                                                                       \
            if (two) {                                                                                 \
                if ((a).wide) hipLaunchKernelGGL((__VA_ARGS__, true, true>), g, b, 0, st, a);          \
                else hipLaunchKernelGGL((__VA_ARGS__, false, true>), g, b, 0, st, a);                  \
                break;                                                                                 \
            }                                                                                          \
        }                                                                                              \
        if ((a).wide) hipLaunchKernelGGL((__VA_ARGS__, true, false>), g, b, 0, st, a);                 \
        else hipLaunchKernelGGL((__VA_ARGS__, false, false>), g, b, 0, st, a);                         \
    } while (0)
template <int NP, int DP>
void launch_fwd(const AttnArgs &a, bool two, int64_t blocks, hipStream_t st)
{
    const dim3 g((unsigned)blocks), b(NT);
    MVF_ATTN_LAUNCH(two, g, b, st, a, k_attn_fwd<NP, DP, tile_states(NP, DP));
}
template <int NP, int DP, int ROWS>
void launch_few_rows(const AttnArgs &a, bool two, int64_t blocks, hipStream_t st)
{
    const dim3 g((unsigned)blocks), b(64 * few_waves_of(NP, DP, ROWS));
    MVF_ATTN_LAUNCH(two, g, b, st, a, k_attn_few<NP, DP, ROWS);
}
template <int NP, int DP>
void launch_few(const AttnArgs &a, bool two, int rows, int64_t blocks, hipStream_t st)
{
    if (rows == 16) launch_few_rows<NP, DP, 16>(a, two, blocks, st);
    else launch_few_rows<NP, DP, 32>(a, two, blocks, st);
}
template <int NP, int DP>
void launch_dq(const AttnArgs &a, int64_t blocks, hipStream_t st)
{
    constexpr int BT = tile_states(NP, DP);
    if (a.wide) hipLaunchKernelGGL((k_attn_dq<NP, DP, BT, true>), dim3((unsigned)blocks), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((k_attn_dq<NP, DP, BT, false>), dim3((unsigned)blocks), dim3(NT), 0, st, a);
}
template <int NP, int DP>
void launch_dkv(const AttnArgs &a, bool two, int64_t blocks, hipStream_t st)
{
    const dim3 g((unsigned)blocks), b(NT);
    MVF_ATTN_LAUNCH(two, g, b, st, a, k_attn_dkv<NP, DP, tile_rows(NP, DP));
}
template <int MODE>
void launch_join(const AttnArgs &a, int NP, int64_t rows, hipStream_t st)
{
    int per = 1;
    while (per * 4 < a.D) per *= 2;
    if (a.splits <= kFlat) {
        const dim3 g((unsigned)((rows + NT / per - 1) / (NT / per)));
        if (NP == 1) hipLaunchKernelGGL((k_attn_join_flat<__bf16, MODE>), g, dim3(NT), 0, st, a, per, rows);
        else hipLaunchKernelGGL((k_attn_join_flat<float, MODE>), g, dim3(NT), 0, st, a, per, rows);
        return;
    }
    const int wpr = rows <= 4 * kCUs ? NT / 64 : 1, rpb = NT / 64 / wpr;
    const dim3 g((unsigned)((rows + rpb - 1) / rpb));
    if (NP == 1) hipLaunchKernelGGL((k_attn_join<__bf16, MODE>), g, dim3(NT), 0, st, a, per, wpr, rows);
    else hipLaunchKernelGGL((k_attn_join<float, MODE>), g, dim3(NT), 0, st, a, per, wpr, rows);
}
#define MVF_ATTN_PICK(fn, p, ...)                                                                      \
    do {                                                                                               \
        if ((p).NP == 1) {                                                                             \
            if ((p).DP == 32) fn<1, 32>(__VA_ARGS__);                                                  \
            else if ((p).DP == 64) fn<1, 64>(__VA_ARGS__);                                             \
            else if ((p).DP == 96) fn<1, 96>(__VA_ARGS__);                                             \
            else fn<1, 128>(__VA_ARGS__);                                                              \
        } else {                                                                                       \
            if ((p).DP == 32) fn<3, 32>(__VA_ARGS__);                                                  \
            else if ((p).DP == 64) fn<3, 64>(__VA_ARGS__);                                             \
            else if ((p).DP == 96) fn<3, 96>(__VA_ARGS__);                                             \
            else fn<3, 128>(__VA_ARGS__);                                                              \
        }                                                                                              \
    } while (0)

int64_t tensor_bytes(const mvf_attn_desc &d, int64_t rows) { return rows * d.D * (d.dtype == MVF_DTYPE_F32 ? 4 : 2); }

}  // namespace

extern "C" {

size_t mvf_cross_attention_fwd_workspace_bytes(const mvf_attn_desc *d)
{
    if (bad_desc(d)) return 0;
    const Plan p = plan_of(*d);
    const int64_t rows = (int64_t)d->B * d->Hq * d->Lq;
    return p.fs > 1 ? (size_t)(p.fs * rows * (d->D + 2) * 4) : 0;
}

int mvf_cross_attention_fwd(const mvf_attn_desc *d, void *out, float *lse, void *workspace, void *stream)
{
    if (bad_desc(d)) return (int)hipErrorInvalidValue;
    if (d->B == 0 || d->Lq == 0) return 0;
    const Plan p = plan_of(*d);
    if (!d->q || !out || (d->Lk > 0 && (!d->k || !d->v)) || (p.fs > 1 && !workspace) || (((uintptr_t)out | (uintptr_t)d->out_low | (uintptr_t)workspace) & 15))
        return (int)hipErrorInvalidValue;
    AttnArgs a = args_of(*d, p);
    const int64_t rows = (int64_t)d->B * d->Hq * d->Lq;
    a.out = out;
    a.lse = lse;
    a.tiles = p.rtiles; a.splits = p.fs; a.per = p.fper;
    a.part = (float *)workspace;
    a.part2 = p.fs > 1 ? a.part + p.fs * rows * d->D : nullptr;
    hipStream_t st = (hipStream_t)stream;
    ProfScope ps(MVF_PROF_ATTN_FWD, st, tensor_bytes(*d, 2 * rows + 2LL * d->B * d->Hk * d->Lk));
    if (p.few) MVF_ATTN_PICK(launch_few, p, a, p.two_f, p.few, (int64_t)d->B * d->Hk * p.fs, st);
    else MVF_ATTN_PICK(launch_fwd, p, a, p.two_f, (int64_t)d->B * d->Hk * p.rtiles * p.fs, st);
    if (p.fs > 1) launch_join<0>(a, p.NP, rows, st);
    return hip_check_launch();
}

size_t mvf_cross_attention_bwd_workspace_bytes(const mvf_attn_desc *d)
{
    if (bad_desc(d)) return 0;
    const Plan p = plan_of(*d);
    const int64_t rows = (int64_t)d->B * d->Hq * d->Lq, states = (int64_t)d->B * d->Hk * d->Lk;
    const int64_t delta = (rows + 3) / 4 * 4;
    const int64_t pq = p.qs > 1 ? p.qs * rows * d->D : 0, pk = p.ks > 1 ? 2 * p.ks * states * d->D : 0;
    return (size_t)((delta + (pq > pk ? pq : pk)) * 4);
}

int mvf_cross_attention_bwd(const mvf_attn_desc *d, const void *out, const float *lse, const void *g_out, void *g_q, void *g_k,
                            void *g_v, void *workspace, void *stream)
{
    if (bad_desc(d)) return (int)hipErrorInvalidValue;
    if (d->B == 0) return 0;
    if (d->Lq > 0 && (!d->q || !out || !lse || !g_out || !g_q || !workspace)) return (int)hipErrorInvalidValue;
    if (d->Lk > 0 && (!d->k || !d->v || !g_k != !g_v)) return (int)hipErrorInvalidValue;
    if (((uintptr_t)out | (uintptr_t)d->out_low | (uintptr_t)g_out | (uintptr_t)g_q | (uintptr_t)g_k | (uintptr_t)g_v | (uintptr_t)workspace) & 15)
        return (int)hipErrorInvalidValue;
    const Plan p = plan_of(*d);
    AttnArgs a = args_of(*d, p);
    const int64_t rows = (int64_t)d->B * d->Hq * d->Lq, states = (int64_t)d->B * d->Hk * d->Lk;
    a.o = out; a.go = g_out; a.lse = const_cast<float *>(lse);
    a.dq = g_q; a.dk = g_k; a.dv = g_v;
    a.delta = (float *)workspace;
    a.part = a.delta + (rows + 3) / 4 * 4;
    hipStream_t st = (hipStream_t)stream;
    ProfScope ps(MVF_PROF_ATTN_BWD, st, tensor_bytes(*d, 4 * rows + 4 * states));
    if (d->Lq > 0) {
        a.tiles = p.rtiles; a.splits = p.qs; a.per = p.qper;
        MVF_ATTN_PICK(launch_dq, p, a, (int64_t)d->B * d->Hk * p.rtiles * p.qs, st);
        if (p.qs > 1) launch_join<1>(a, p.NP, rows, st);
    }
    if (d->Lk > 0 && g_k) {
        a.tiles = p.ktiles; a.splits = p.ks; a.per = p.kper;
        MVF_ATTN_PICK(launch_dkv, p, a, p.two_k, (int64_t)d->B * d->Hk * p.ktiles * p.ks, st);
        if (p.ks > 1) launch_join<2>(a, p.NP, 2 * states, st);
    }
    return hip_check_launch();
}

}  // extern "C"
