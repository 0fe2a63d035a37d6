// ssm.hip -- operators of a state-space language-model block over packed residue rows: short causal convolution, selective scan, both for one
// token, and the norms around the block (include/mdfri.h "Operators of a state-space language-model block").
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace mdf {

typedef unsigned short u16;

struct F16 {
    u16 v;
};
struct Bf16 {
    u16 v;
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(Bf16 x) { return __uint_as_float((unsigned)x.v << 16); }
__device__ __forceinline__ float to_f32(F16 x) { return (float)__builtin_bit_cast(_Float16, x.v); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ Bf16 from_f32<Bf16>(float x) { return {__builtin_bit_cast(u16, (__bf16)x)}; }   // round to nearest even
template <> __device__ __forceinline__ F16 from_f32<F16>(float x) { return {__builtin_bit_cast(u16, (_Float16)x)}; }

// v_rcp_f32 is within one step: an IEEE division is ten instructions per value, and these run once per element of arrays that stream from memory
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }
__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }
// max(v, 0) + log(1 + t), t = e^-|v|; log(1 + t) = 2 artanh(s) with s = t / (2 + t) <= 1/3, its series to s^15 (the rest is below 2^-26 of it)
__device__ __forceinline__ float softplus(float v)
{
    const float t = __expf(-fabsf(v)), s = t * __builtin_amdgcn_rcpf(2.0f + t), q = s * s;
    float r = fmaf(q, 2.0f / 15.0f, 2.0f / 13.0f);
    r = fmaf(q, r, 2.0f / 11.0f);
    r = fmaf(q, r, 2.0f / 9.0f);
    r = fmaf(q, r, 2.0f / 7.0f);
    r = fmaf(q, r, 2.0f / 5.0f);
    r = fmaf(q, r, 2.0f / 3.0f);
    r = fmaf(q, r, 2.0f);
    return fmaf(s, r, v > 0.0f || v != v ? v : 0.0f);   // (a NaN stays one, -infinity gives 0)
}
// one value of any of the three types, by code (uniform): the step sizes dt, which are read once per head and row
__device__ __forceinline__ float load_any(const void *p, size_t i, int dt)
{
    return dt == MDF_DT_F32 ? static_cast<const float *>(p)[i] : dt == MDF_DT_BF16 ? to_f32(static_cast<const Bf16 *>(p)[i]) : to_f32(static_cast<const F16 *>(p)[i]);
}

// N values as they lie in memory: one 16-byte access (f32: two for 8) at whatever alignment the values themselves have -- the global memory path takes
// any address, at the price of one more cache line where an access crosses one, so odd strides and views need no code of their own
template <typename T, int N>
struct Raw {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T *p)
{
    Raw<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_raw(T *p, const Raw<T, N> &r)
{
    __builtin_memcpy(p, &r, sizeof(r));
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T *p, const float *v)
{
    Raw<T, N> r;
    if constexpr (std::is_same<T, Bf16>::value && N % 2 == 0) {   // one conversion for two values
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        unsigned u[N / 2];
#pragma unroll
        for (int i = 0; i < N; i += 2) u[i / 2] = __builtin_bit_cast(unsigned, __builtin_convertvector((f2){v[i], v[i + 1]}, b2));
        __builtin_memcpy(&r, u, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(v[i]);
    }
    store_raw(p, r);
}

// What a kernel knows of a sequence; count < 0: skipped (its slot is outside the pool, or it has no rows)
struct Seq {
    int64_t row;      // first row
    int count;        // rows to work on
    int rows;         // rows
    int slot;
    int64_t pos;      // tokens before
};
__device__ __forceinline__ Seq seq_of(const mdf_seq_rows &r, int b, bool kept)
{
    Seq s;
    s.row = r.row_off[b];
    int64_t n = r.lengths[b];
    if (s.row < 0 || s.row > r.R) n = 0;
    n = n < 0 ? 0 : n > r.R - s.row ? r.R - s.row : n;
    s.count = s.rows = (int)n;
    s.slot = kept && r.slots ? r.slots[b] : b;
    s.pos = kept && r.positions ? r.positions[b] : 0;
    if (s.pos < 0) s.pos = 0;
    if (kept && (s.slot < 0 || s.slot >= r.n_slots)) s.count = -1;
    return s;
}
// The last sequence that begins at or before `row` (row_off ascends), or -1.
__device__ __forceinline__ int seq_before(const int32_t *row_off, int B, int64_t row)
{
    int lo = -1, hi = B;   // row_off[lo] <= row < row_off[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (row_off[m] <= row) lo = m; else hi = m;
    }
    return lo;
}

// ---- the short causal convolution ----------------------------------------------------------------------------------------------------------------
// A thread owns V channels (16 bytes) of `steps` tiles of CONV_ROWS rows.  A tile's rows are requested at once, the width - 1 in front of them are still
// in registers from the tile before (or requested too), the weights stay in registers.  Bound by memory: each element is read and written once
// (144 753 rows x 640 in 256 sequences, width 4, bfloat16: 371 MB in 93 us, 4.0 TB/s; SiLU and the conversions are about 17 instructions a value under it).  Tiles of
// 16 rows or 4 channels a thread measured 100 to 232 us there.
// Rows take their taps from registers; only a sequence's first width - 1 rows, which look into the kept state or before the sequence, look
// every tap up.  The tile with a sequence's first row makes all of those rows, wherever they lie, and then keeps the sequence's last inputs:
// nobody else reads or writes these channels' entries, so a short sequence that overwrites an entry it still needed is no race.
constexpr int CONV_ROWS = 8;

template <typename T, int V, int W>
__global__ __launch_bounds__(256, W <= 3 ? 3 : W <= 7 ? 2 : 1) void k_conv(mdf_conv_args g, int steps, int lanes)   // lanes = channels / V, rounded up; channels >= V
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t tile0 = id / lanes * steps;
    // The last lane of an uneven row is moved up against the row's end: it makes `twice` channels that its neighbour makes too, to the same bits -- but
    // for a sequence's first rows, whose kept inputs the neighbour may have replaced already, it stores its own channels only.
    const int c = min((int)(id % lanes) * V, g.channels - V), twice = (int)(id % lanes) * V - c;
    if (tile0 * CONV_ROWS >= g.rows.R) return;
    Raw<float, V> w[W], bias = {};
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = load_raw<float, V>(g.weight + (size_t)k * g.channels + c);
    if (g.bias) bias = load_raw<float, V>(g.bias + c);
    const T *x = static_cast<const T *>(g.x) + c;
    T *out = static_cast<T *>(g.out) + c, *ring = static_cast<T *>(g.state) + c;
    int b = seq_before(g.rows.row_off, g.rows.B, tile0 * CONV_ROWS);
    Seq s = {0, -1, 0, 0, 0};
    int64_t next;   // first row of the sequence behind s
    auto begin = [&]() {
        if (b >= 0) s = seq_of(g.rows, b, g.state != nullptr);
        next = b + 1 < g.rows.B ? g.rows.row_off[b + 1] : g.rows.R;
    };
    begin();
    Raw<T, V> raw[CONV_ROWS + W - 1];
    for (int step = 0; step < steps; ++step) {
        const int64_t r0 = (tile0 + step) * CONV_ROWS, r1 = min(r0 + CONV_ROWS, g.rows.R);
        if (r0 >= r1) return;
        unsigned mask = (1u << CONV_ROWS) - 1;   // rows whose taps are all in registers
        if (!(r0 - s.row >= max(W - 1, 1) && r0 + CONV_ROWS - s.row <= s.count)) {   // (the next sequence begins behind this one's rows)
            auto row = [&](int t) {   // one of a sequence's first rows
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = bias.v[i];
#pragma unroll
                for (int back = W - 1; back >= 0; --back) {
                    Raw<T, V> u = {};
                    if (t >= back) u = load_raw<T, V>(x + (size_t)(s.row + t - back) * g.ldx);
                    else if (g.state && s.pos + t >= back) u = load_raw<T, V>(ring + ((size_t)s.slot * W + (size_t)((s.pos + t - back) % W)) * g.channels);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = fmaf(w[W - 1 - back].v[i], to_f32(u.v[i]), v[i]);
                }
                T *o = out + (size_t)(s.row + t) * g.ldo;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i >= twice) o[i] = from_f32<T>(g.silu ? silu(v[i]) : v[i]);
            };
            auto finish = [&](int from) {   // the first rows from `from` on, then the sequence's last inputs into its state
                for (int t = from; t < min(s.count, W - 1); ++t) row(t);
                if (!g.state) return;
                Raw<T, V> last[W];
#pragma unroll
                for (int k = 0; k < W; ++k) last[k] = load_raw<T, V>(x + (size_t)(s.row + max(s.count - W + k, 0)) * g.ldx);
#pragma unroll
                for (int k = 0; k < W; ++k)
                    if (s.count - W + k >= 0) {
                        T *entry = ring + ((size_t)s.slot * W + (size_t)((s.pos + s.count - W + k) % W)) * g.channels;
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            if (i >= twice) entry[i] = last[k].v[i];
                    }
            };
            mask = 0;
            for (int64_t r = r0; r < r1; ++r) {
                while (r >= next) ++b, begin();
                const int64_t t = r - s.row;
                if (b >= 0 && s.count < 0 && t < s.rows && g.zero_skipped) {
                    const float zero[V] = {};
                    store_f32<T, V>(out + (size_t)r * g.ldo, zero);
                }
                if (b < 0 || t >= s.count) continue;
                if (t == 0) finish(0);
                if (t >= W - 1) mask |= 1u << (int)(r - r0);
            }
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) raw[k] = step ? raw[CONV_ROWS + k] : load_raw<T, V>(x + (size_t)max(r0 - (W - 1) + k, (int64_t)0) * g.ldx);
#pragma unroll
        for (int k = 0; k < CONV_ROWS; ++k) raw[W - 1 + k] = load_raw<T, V>(x + (size_t)min(r0 + k, g.rows.R - 1) * g.ldx);
        auto make = [&](int r) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = bias.v[i];
#pragma unroll
                for (int k = 0; k < W; ++k) v[i] = fmaf(w[k].v[i], to_f32(raw[r + k].v[i]), v[i]);
                if (g.silu) v[i] = silu(v[i]);
            }
            store_f32<T, V>(out + (size_t)(r0 + r) * g.ldo, v);
        };
        if (mask == (1u << CONV_ROWS) - 1) {
#pragma unroll
            for (int r = 0; r < CONV_ROWS; ++r) make(r);
        } else {
#pragma unroll
            for (int r = 0; r < CONV_ROWS; ++r)
                if (mask >> r & 1) make(r);
        }
    }
}

// ---- the selective scan ----------------------------------------------------------------------------------------------------------------------------
// Chunks of 32 rows.  With c_i the running log-decay inside a chunk (c_i <= 0, base 2), S the state in front of it and D_j the step sizes, the recurrence is
//     Y = diag(2^c_i) (C S)  +  M X + d X,      M_ij = (C_i . B_j) 2^(c_i - c_j) D_j  for j <= i, 0 above
//     S <- 2^c_31 S + B^T diag(D_j 2^(c_31 - c_j)) X
// -- four products on the bf16 matrix instruction (32 x 32 x 16), all sums and the state in f32.  A wave owns 32 channels of a head and their whole
// state (16 registers per 32 state values); four waves of a workgroup, channels of the same group of heads, share the chunk's B and C in LDS.
// No operand goes through LDS on its way from one product to the next: result registers hold, per lane half, four consecutive rows in the very place where
// the next product takes them as its k.  For M that order is 0-3, 8-11 | 4-7, 12-15 per 16, and X is read in it; the state's rows are put in such an order by
// the reads of B^T that its registers are k in their natural order and C is read as it lies.  (B C^T) comes out transposed,
// lane = i, and so does Y: a lane holds four consecutive channels of a row, which leave in 16-byte stores (with a swap between the halves for 16-bit types).
// X comes in 16-byte loads through a tile in LDS; it and B^T are read from their rows by the transposing read.
// Operands are sums of bfloat16 terms: bfloat16 inputs are one, float16 two and float32, M, S and what goes into the state three (all exact).  Of the term products
// of two such sums those below 2^-24 are left out -- none where one of the two is bfloat16; elsewhere the second of three terms is rounded, so that what is left out
// has no sign of its own (48 float32 sequences, off 64 bits: 1.32e-7 -> 1.19e-7 in the same time; two more products give 1.19e-7 too, in 9 % more).  So for
// every type the arithmetic is that of float32, and a 16-bit output is rounded once.  (M and S in two terms, 2^-16, took 324 us in place of 360 in the case
// below, and left its bfloat16 outputs 1.2e-4 in the 2-norm off those of float32 products; now 2.3e-5.)
// Bound for bfloat16 by work that hardly overlaps with two waves per SIMD: per chunk and wave about 980 vector and 62 matrix instructions (state_dim 128) and the
// rows of X and Y.  128 sequences of 512 rows, 32 heads of 64 x 128: 346 to 360 us from card to card (its bytes would take 113); 263 without the matrix instructions,
// 303 without splitting S, M and W into terms, 270 without loading X and storing Y.  Some of it is made more than once: G = B C^T by each of the four waves (8 of the
// 62), M by both waves of a 64-channel head.  float16 takes 650 there, float32 850: one wave per SIMD.
// Measured with two terms of S and M, at 319 to 337: 8 waves a workgroup 335, three waves per SIMD 590 (spills), matrix and vector instructions woven by hand 346.
// Long sequences are cut into segments when there are too few (sequence, head) pairs to fill the GPU: a first launch makes each segment's state from zero
// (STATE: no Y, no C), a small one carries the states from segment to segment, the last one makes Y.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ unsigned cvt_pk_bf16(float a, float b)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, b2));
}
// Two values -> TERMS packed bf16 pairs whose sum they are: each term takes the leading 8 bits of what the ones before leave over (cut off, not rounded:
// one v_perm for the pair), so three terms are exact for float32, two for float16.  ROUND: the second of three is rounded to nearest (a conversion for the pair, and
// no overflow as there would be with the first): the third, exact still, is half as large and of either sign, and so are the products of terms that are left out.
template <int TERMS, bool ROUND = false>
__device__ __forceinline__ void split_pair(float a, float b, unsigned (&o)[TERMS])
{
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        if (ROUND && TERMS == 3 && i == 1) {
            o[i] = cvt_pk_bf16(a, b);
            a -= __uint_as_float(o[i] << 16);
            b -= __uint_as_float(o[i] & 0xffff0000u);
            continue;
        }
        o[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);   // the upper halves
        if (i + 1 < TERMS) {
            a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
            b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        }
    }
}
template <int TERMS, bool ROUND = false>
__device__ __forceinline__ void split8(const float *v, u32x4 (&o)[TERMS])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned u[TERMS];
        split_pair<TERMS, ROUND>(v[2 * i], v[2 * i + 1], u);
#pragma unroll
        for (int k = 0; k < TERMS; ++k) o[k][i] = u[k];
    }
}
// acc += a . b over the term pairs (i, j), i + j <= MOST, smallest first
template <int MOST, int LA, int LB>
__device__ __forceinline__ void product(f32x16 &acc, const u32x4 (&a)[LA], const u32x4 (&b)[LB])
{
#pragma unroll
    for (int s = MOST; s >= 0; --s)
#pragma unroll
        for (int i = LA - 1; i >= 0; --i)
            if (s - i >= 0 && s - i < LB)
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[i]), __builtin_bit_cast(bf16x8, b[s - i]), acc, 0, 0, 0);
}

// A lane's 16 values of X -- one channel, rows 8 (i / 4) + 4 half + i % 4 -- out of the wave's tile in LDS, and as the terms of a product operand.  16-bit
// types come four rows at a time by the transposing read: 16 lanes read 4 rows x 16 columns and each gets one column's 4 rows.
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <bool SWAP = false>   // the second and third four of the 16 columns exchanged
__device__ __forceinline__ u32x2 read_columns(const void *tile, int stride, int row, int column)   // rows row .. row + 3, 16 columns from `column` on, over 16 lanes
{
    const int l16 = threadIdx.x & 15, four = SWAP ? (l16 & 1) << 1 | (l16 >> 1 & 1) : l16 & 3;
    const u16 *at = static_cast<const u16 *>(tile) + (row + (l16 >> 2)) * stride + column + 4 * four;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)const_cast<u16 *>(at)));
}
template <typename T> struct Chunk {   // float
    float v[16];
    __device__ __forceinline__ void take(const T *tile, int stride, int half, int l32)
    {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = tile[(8 * (i / 4) + 4 * half + i % 4) * stride + l32];
    }
    __device__ __forceinline__ bool finite(int i) const { return fabsf(v[i]) < __builtin_inff(); }
    __device__ __forceinline__ void clear(int i) { v[i] = 0.0f; }
    __device__ __forceinline__ float get(int i) const { return v[i]; }
    template <int N> __device__ __forceinline__ void terms(int kb, u32x4 (&o)[N]) const { split8<N, true>(v + 8 * kb, o); }
};
template <typename T> struct Packed {   // pairs of 16-bit values
    u32x4 v[2];
    __device__ __forceinline__ void take(const T *tile, int stride, int half, int l32)
    {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const u32x2 u = read_columns(tile, stride, 8 * q + 4 * half, l32 & 16);
            v[q / 2][2 * (q & 1)] = u[0], v[q / 2][2 * (q & 1) + 1] = u[1];
        }
    }
    __device__ __forceinline__ void clear(int i) { v[i / 8][i % 8 / 2] &= i & 1 ? 0xffffu : 0xffff0000u; }
    __device__ __forceinline__ float get(int i) const { return to_f32(T{(u16)(i & 1 ? v[i / 8][i % 8 / 2] >> 16 : v[i / 8][i % 8 / 2])}); }
    __device__ __forceinline__ bool finite(int i) const { return fabsf(get(i)) < __builtin_inff(); }
};
template <> struct Chunk<Bf16> : Packed<Bf16> {   // the pairs are the operand
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i & 1 ? v[i / 8][i % 8 / 2] & 0xffff0000u : v[i / 8][i % 8 / 2] << 16); }
    template <int N> __device__ __forceinline__ void terms(int kb, u32x4 (&o)[N]) const { o[0] = v[kb]; }
};
template <> struct Chunk<F16> : Packed<F16> {
    template <int N> __device__ __forceinline__ void terms(int kb, u32x4 (&o)[N]) const
    {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = get(8 * kb + e);
        split8<N>(f, o);
    }
};
// whether one of 8 values is an infinity or a NaN
__device__ __forceinline__ bool any_odd(const Raw<float, 8> &r)
{
    int most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_int(r.v[i]) & 0x7fffffff);
    return most >= 0x7f800000;
}
template <typename T>
__device__ __forceinline__ bool any_odd(const Raw<T, 8> &r)
{
    typedef u16 h2 __attribute__((ext_vector_type(2)));
    h2 most = {0, 0};
    unsigned u[4];
    __builtin_memcpy(u, &r, sizeof(u));
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(h2, u[i] & 0x7fff7fffu));
    return max(most[0], most[1]) >= (std::is_same<T, Bf16>::value ? 0x7f80 : 0x7c00);
}

// terms of an input, and the largest i + j of the term products of two inputs (float16: all four)
template <typename T> struct Terms;
template <> struct Terms<Bf16> { static constexpr int X = 1, IN = 0; };
template <> struct Terms<F16> { static constexpr int X = 2, IN = 2; };
template <> struct Terms<float> { static constexpr int X = 3, IN = 2; };

constexpr int SCAN_Q = 32, SCAN_WAVES = 4;
constexpr unsigned GRID_X = 1u << 23;   // most workgroups of 256 threads in a launch's x: a dimension of a grid holds fewer than 2^32 threads

// A value the compiler may not compute with ahead of here: what is derived from it in a loop (offsets, comparisons) is made where it is used, one instruction
// each, instead of being kept in dozens of registers over the loop
__device__ __forceinline__ unsigned fresh(unsigned v)
{
    asm volatile("" : "+v"(v));
    return v;
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double v)   // another lane's value; 0 where there is none or the row is not in ROWS
{
    const long long u = __builtin_bit_cast(long long, v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}
__device__ __forceinline__ double lane_f64(double v, int lane)
{
    const long long u = __builtin_bit_cast(long long, v);
    return __builtin_bit_cast(double, (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(u >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)u, lane)));
}

// Raw buffer descriptors: an access whose byte offset lies at or behind the end is dropped, a load gives 0.
constexpr unsigned OUTSIDE = 0x80000000u;   // an offset behind every descriptor made here, with room for the rows that are added to it
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void *p, int rows, unsigned stride, unsigned width)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)((rows - 1) * stride + width), 0x00020000);
}
__device__ __forceinline__ void buffer_load(float &v, __amdgpu_buffer_rsrc_t r, unsigned at) { v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0)); }
__device__ __forceinline__ void buffer_load(Bf16 &v, __amdgpu_buffer_rsrc_t r, unsigned at) { v.v = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0); }
__device__ __forceinline__ void buffer_load(F16 &v, __amdgpu_buffer_rsrc_t r, unsigned at) { v.v = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0); }
__device__ __forceinline__ void buffer_store(float v, __amdgpu_buffer_rsrc_t r, unsigned at) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, at, 0, 0); }
__device__ __forceinline__ void buffer_store(Bf16 v, __amdgpu_buffer_rsrc_t r, unsigned at) { __builtin_amdgcn_raw_buffer_store_b16(v.v, r, at, 0, 0); }
__device__ __forceinline__ void buffer_store(F16 v, __amdgpu_buffer_rsrc_t r, unsigned at) { __builtin_amdgcn_raw_buffer_store_b16(v.v, r, at, 0, 0); }

// Segments of long sequences; rows == 0: none.  A sequence of more than `rows` rows has a slot per segment, from number row / (rows / 2) on, `row` its first:
// its n segments span more than n - 1 times `rows`, so twice as many halves as it has whole segments, no fewer than n, lie in front of the next sequence's first slot.
// So 2 R / rows slots do for any mix of lengths (a shorter sequence has none), and a slot's owner is the last sequence whose slots would begin at or before it.
struct ScanSplit {
    int rows, slots;        // rows per segment (multiple of 64)
    float *states;          // (slots, heads, head_dim, state_dim): a segment's own end state, then its start state
    float *decays;          // (slots, heads): log2 of a segment's whole decay
};
__device__ __forceinline__ int slot_owner(const mdf_seq_rows &r, const ScanSplit &cut, int slot) { return seq_before(r.row_off, r.B, (int64_t)(slot + 1) * (cut.rows / 2) - 1); }

// WORDS: every row of x, b and c, and every head's and group's part of it, begins on a word.  A template, since the choice inside the loop cost aligned calls 375 us
// in place of 319 (128 x 512 rows as above, two terms of S and M); unaligned ones load whole words and shift them.
template <typename T, int NT, bool STATE, bool WORDS>
__global__ __launch_bounds__(64 * SCAN_WAVES, Terms<T>::X > 1 && NT > 2 ? 1 : 2) void k_scan(mdf_scan_args g, ScanSplit cut, int items, int unit_blocks)
{
    typedef Terms<T> K;
    constexpr int TX = K::X, NS = 32 * NT + 8, PS = sizeof(T) == 4 ? 36 : 40, BUF = TX == 1 ? 2 : 1;   // row strides in LDS: a little more than the rows, over the banks
    __shared__ __align__(16) u16 Cs[STATE ? 1 : BUF][STATE ? 1 : TX][SCAN_Q][NS], Bs[BUF][TX][SCAN_Q][NS];
    __shared__ __align__(16) T Xs[SCAN_WAVES][SCAN_Q][PS];
    __shared__ __align__(16) float steps[SCAN_WAVES][2][6][SCAN_Q];   // k = c - log2 D, c, low part of k, D 2^(c_31 - c), 2^c, low part of c, of two chunks
    // Block -> (item, channels): workgroups of one item (which read the same B and C) lie on one XCD -- block b runs on XCD b mod 8 -- and close in time.
    const int xcd = blockIdx.x & 7, place = (int)(blockIdx.y * (GRID_X / 8) + (blockIdx.x >> 3)), item = (place / unit_blocks) * 8 + xcd, ub = place % unit_blocks;
    if (item >= items) return;
    // items: the slots of segments, then the sequences that are not cut
    const int b = item >= cut.slots ? item - cut.slots : __builtin_amdgcn_readfirstlane(slot_owner(g.rows, cut, item));
    if (b < 0) return;
    Seq s = seq_of(g.rows, b, g.state != nullptr);
    s.row = __builtin_amdgcn_readfirstlane((int)s.row), s.count = __builtin_amdgcn_readfirstlane(s.count);   // the same in every lane: addresses by the scalar unit
    const bool split = cut.rows && s.count > cut.rows;
    const int slot0 = split ? (int)s.row / (cut.rows / 2) : 0, seg = split ? item - slot0 : 0;
    if (split != (item < cut.slots) || seg < 0 || (split && (int64_t)seg * cut.rows >= s.count)) return;   // another item's sequence, or a slot that no segment has
    const int first = split ? seg * cut.rows : 0;
    if (!STATE && s.count < 0 && g.zero_skipped) {
        const int r = g.heads / g.groups, pblocks = (g.head_dim + 31) / 32, per_group = (r * pblocks + SCAN_WAVES - 1) / SCAN_WAVES, h0 = ub / per_group * r;
        const int u0 = ub % per_group * SCAN_WAVES, u1 = min(u0 + SCAN_WAVES, r * pblocks) - 1;   // the workgroup's channels lie side by side
        const int c0 = (h0 + u0 / pblocks) * g.head_dim + u0 % pblocks * 32, c1 = (h0 + u1 / pblocks) * g.head_dim + min(u1 % pblocks * 32 + 32, g.head_dim);
        for (int t = 0; t < s.rows; ++t)
            for (int c = c0 + threadIdx.x; c < c1; c += 64 * SCAN_WAVES) static_cast<T *>(g.y)[(size_t)(s.row + t) * g.ldy + c] = from_f32<T>(0.0f);
    }
    if (s.count <= 0) return;                                         // skipped, or without rows
    const int last = split ? (int)min((int64_t)first + cut.rows, (int64_t)s.count) : s.count;
    if (STATE && last == s.count) return;                              // nobody starts from this segment's end
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l32 = lane & 31;
    const int N = g.state_dim, P = g.head_dim, r = g.heads / g.groups, pblocks = (P + 31) / 32, per_group = (r * pblocks + SCAN_WAVES - 1) / SCAN_WAVES;
    const int grp = ub / per_group, unit = (ub % per_group) * SCAN_WAVES + wave;
    const bool works = unit < r * pblocks;                             // the others help with B and C
    const int h = works ? grp * r + unit / pblocks : grp * r, p = (unit % pblocks) * 32 + l32;
    const bool mine = works && p < P;
    const size_t row0 = (size_t)s.row;
    const float a = g.a[h], bias = g.dt_bias ? g.dt_bias[h] : 0.0f, skip = g.d ? g.d[h] : 0.0f;

    // the state: register i of tile nt is n = 32 nt + 16 (i / 8) + 8 half + i % 8 of channel p
    f32x16 S[NT];
    const size_t head = (size_t)h * P * N, seg_cells = (size_t)g.heads * P * N;
    const float *start = split ? (STATE ? nullptr : cut.states + (size_t)(slot0 + seg) * seg_cells) : g.state && s.pos > 0 ? g.state + (size_t)s.slot * seg_cells : nullptr;
    float *end = STATE ? cut.states + (size_t)(slot0 + seg + 1) * seg_cells : g.state && last == s.count ? g.state + (size_t)s.slot * seg_cells : nullptr;
    auto cell = [&](int n) { return mine && n < N ? fresh((unsigned)(p * N) * 4u) + 4u * n : OUTSIDE; };   // inside the head's state
    if (start && works) {
        const auto sr = rows_at(start + head, 1, 0, (unsigned)(P * N) * 4u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = 32 * nt + 16 * (q >> 1) + 8 * half + 4 * (q & 1);
                if ((N & 3) == 0) {
                    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(sr, cell(n), 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[nt][4 * q + e] = __uint_as_float(v[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[nt][4 * q + e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sr, cell(n + e), 0, 0));
                }
            }
    } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] = f32x16{};
    }
    double total = 0.0;                                                // log2 of the decay since `first` (STATE)

    // What the next chunk needs, on its way from memory, 8 values each: PER times of B and C, twice of the wave's 32 columns of X; the step sizes of two chunks.
    // All through buffer descriptors that end with the chunk's last row: rows behind it read as 0 and are not written.
    constexpr int PER = (NT + 1) / 2;
    constexpr unsigned E = sizeof(T);
    const int p0 = unit % pblocks * 32;
    const unsigned xrow = (unsigned)g.ldx * E, yrow = (unsigned)g.ldy * E, brow = (unsigned)g.ldb * E, crow = (unsigned)g.ldc * E, width = (unsigned)(g.heads * P) * E;
    const unsigned col = (unsigned)(h * P + p0) * E;
    const char *bp = static_cast<const char *>(g.b) + row0 * brow + (size_t)grp * N * E, *cp = static_cast<const char *>(g.c) + row0 * crow + (size_t)grp * N * E;
    const char *xp = static_cast<const char *>(g.x) + row0 * xrow;
    char *yp = static_cast<char *>(g.y) + row0 * yrow;
    auto words = [](const void *q, unsigned row) { return ((reinterpret_cast<uintptr_t>(q) | row) & 3) == 0; };   // buffer accesses want addresses of whole words
    const bool ywide = words(yp, yrow) && P % (sizeof(T) == 4 ? 4 : 8) == 0;
    // 8 values on their way.  Where rows or bases begin inside a word (16-bit types), the five words around them; `settle`, once they are there, shifts them into
    // place and clears what lies behind a row's end -- not here: that would wait for the load at once.
    struct Load {
        Raw<T, 8> v;
        unsigned more;
    };
    Load rb[PER] = {}, rc[PER] = {}, rx[2] = {};
    float rdt = 0.0f;
    auto skew = [](const void *q) { return WORDS ? 0u : (unsigned)(reinterpret_cast<uintptr_t>(q) & 3); };
    auto whole = [&](const char *q, int rows, unsigned stride, unsigned bytes) {   // a descriptor over whole words
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(q) - skew(q), 0, (int)(((rows - 1) * stride + bytes + skew(q) + 3) & ~3u), 0x00020000);
    };
    auto fetch8 = [&](Load &l, __amdgpu_buffer_rsrc_t r, unsigned offset, int left) {
        const unsigned at = fresh(left > 0 ? offset : OUTSIDE);
        if constexpr (WORDS) {
            u32x4 u[E / 2];
#pragma unroll
            for (int i = 0; i < (int)E / 2; ++i) u[i] = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * i, 0, 0);
            __builtin_memcpy(&l.v, u, sizeof(l.v));
        } else {
            const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(r, at & ~3u, 0, 0);
            __builtin_memcpy(&l.v, &u, 16);
            l.more = __builtin_amdgcn_raw_buffer_load_b32(r, (at & ~3u) + 16, 0, 0);
        }
    };
    auto settle = [&](Load &l, unsigned offset, int left, bool exact, bool there) {   // `there`: a row of the chunk (its last word may hold the next row's first value)
        if constexpr (!WORDS) {
            if (!there) {
                l.v = {};
                return;
            }
            unsigned u[5];
            __builtin_memcpy(u, &l.v, 16);
            u[4] = l.more;
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __builtin_amdgcn_alignbit(u[i + 1], u[i], (offset & 2) * 8);
            __builtin_memcpy(&l.v, u, 16);
        }
        if (exact)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= left) l.v.v[e] = T{};
    };
    auto request = [&](int t0) {
        if (t0 >= last) return;
        const int rows = min(SCAN_Q, last - t0);
        const char *b0 = bp + (size_t)t0 * brow, *c0 = cp + (size_t)t0 * crow;
        const auto br = whole(b0, rows, brow, N * E), cr = whole(c0, rows, crow, N * E);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = threadIdx.x + 256 * k, row = i / (4 * NT), n = i % (4 * NT) * 8;
            if (128 * NT % 256 && i >= 128 * NT) continue;
            fetch8(rb[k], br, skew(b0) + row * brow + n * E, N - n);
            if (!STATE) fetch8(rc[k], cr, skew(c0) + row * crow + n * E, N - n);
        }
        if (!works) return;
        const char *x0 = xp + (size_t)t0 * xrow;
        const auto xr = whole(x0, rows, xrow, width);
#pragma unroll
        for (int k = 0; k < 2; ++k) fetch8(rx[k], xr, skew(x0) + (lane / 4 + 16 * k) * xrow + col + lane % 4 * 8 * E, P - p0 - lane % 4 * 8);
    };
    auto request_dt = [&](int t0) { rdt = t0 + lane < last ? load_any(g.dt, (row0 + t0 + lane) * g.lddt + h, g.dt_dtype) : 0.0f; };
    // Step sizes and running log-decays of two chunks from t0 on, lanes 0-31 and 32-63; the sum in double: differences of far apart rows keep their bits
    auto decays = [&](int t0) {
        const float D = t0 + lane < last ? softplus(rdt + bias) : 0.0f;
        double c = (double)D * (double)a * 1.4426950408889634;
        c += dpp_f64<0x111>(c);          // from the lane 1, 2, 4, 8 below in its row of 16 (0 from outside it) ...
        c += dpp_f64<0x112>(c);
        c += dpp_f64<0x114>(c);
        c += dpp_f64<0x118>(c);
        c += dpp_f64<0x142, 0xa>(c);     // ... and from lane 15 of the row below, into rows 1 and 3
        const double c31 = half ? lane_f64(c, 63) : lane_f64(c, 31);
        // D_j 2^(c_i - c_j) = 2^(c_i - k_j), k = c - log2 D; D = 0 gives k = infinity and a factor of 0.  The logarithm as v_log and what it is off by; v_log takes a
        // subnormal D for 0, and then 2^-lg is an infinity, which must not meet the one in lg.
        const float lg = __builtin_amdgcn_logf(D);
        const float off = D >= 1.17549435e-38f ? fmaf(D, __builtin_amdgcn_exp2f(-lg), -1.0f) * 1.44269504f : 0.0f;
        const double kd = c - (double)lg - (double)off;
        const float hi = (float)c, khi = (float)kd;
        steps[wave][half][0][l32] = khi;
        steps[wave][half][1][l32] = hi;
        steps[wave][half][2][l32] = isinf(khi) ? 0.0f : (float)(kd - (double)khi);
        steps[wave][half][3][l32] = D * __builtin_amdgcn_exp2f((float)(c31 - c));
        steps[wave][half][4][l32] = __builtin_amdgcn_exp2f(hi);
        steps[wave][half][5][l32] = (float)(c - (double)hi);
        if (STATE) total += lane_f64(c, 31) + lane_f64(c, 63);
        request_dt(t0 + 2 * SCAN_Q);
    };
    // What has arrived into LDS: B and C as terms, X as it is
    bool odd = false;
    auto stage = [&](int buf, int t0) {
        odd = false;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = threadIdx.x + 256 * k, row = i / (4 * NT), n = i % (4 * NT) * 8;
            if (128 * NT % 256 && i >= 128 * NT) continue;
#pragma unroll
            for (int m = 0; m < (STATE ? 1 : 2); ++m) {
                const unsigned stride = m ? crow : brow;
                settle(m ? rc[k] : rb[k], skew((m ? cp : bp) + (size_t)t0 * stride) + row * stride + n * E, N - n, N & 7, t0 + row < last);
                const Raw<T, 8> &v = m ? rc[k].v : rb[k].v;
                u32x4 u[TX];
                if constexpr (TX == 1) __builtin_memcpy(u, &v, 16);
                else {
                    float f[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = to_f32(v.v[e]);
                    split8<TX, true>(f, u);
                }
#pragma unroll
                for (int x = 0; x < TX; ++x) {
                    u16 *to = &Bs[buf][x][row][n];
                    if constexpr (!STATE)
                        if (m) to = &Cs[buf][x][row][n];
                    *reinterpret_cast<u32x4 *>(to) = u[x];
                }
            }
        }
        if (works)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                settle(rx[k], skew(xp + (size_t)t0 * xrow) + (lane / 4 + 16 * k) * xrow + col + lane % 4 * 8 * E, 8, false, t0 + lane / 4 + 16 * k < last);
                odd |= any_odd(rx[k].v);
                __builtin_memcpy(__builtin_assume_aligned(&Xs[wave][lane / 4 + 16 * k][lane % 4 * 8], 16), &rx[k].v, sizeof(rx[k].v));
            }
    };
    // Loads are waited for in the order they and the stores were issued, so a chunk is staged in front of the stores of the one before it: behind them it would
    // wait for their way to memory too, once per chunk (346 -> 337 us, two terms of S and M).
    request(first);
    request_dt(first);
    decays(first);
    stage(0, first);
    request(first + SCAN_Q);
    for (int t0 = first, k = 0; t0 < last; t0 += SCAN_Q, ++k) {
        const int buf = BUF == 2 ? k & 1 : 0;
        const bool spoilt = __any(odd);
        __syncthreads();
        f32x16 Y = {};
        if (works) {
        // ---- X.  A value that is not finite would reach rows in front of it in M X (0 x NaN): it counts as 0, spoils its own and the later rows of its channel by
        // hand, and the channel's state.
        const float(&st)[6][SCAN_Q] = steps[wave][k & 1];
        Chunk<T> xc;
        xc.take(&Xs[wave][0][0], PS, half, l32);
        int bad = SCAN_Q;
        if (spoilt) {
            asm volatile("; a value that is not finite");   // (keeps what follows out of the ordinary path)
#pragma unroll
            for (int i = 15; i >= 0; --i)
                if (!xc.finite(i)) xc.clear(i), bad = 8 * (i / 4) + 4 * half + i % 4;
            bad = min(bad, __shfl_xor(bad, 32));
        }
        u32x4 X[2][TX], W[2][3];
        if constexpr (!STATE) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) xc.terms(kb, X[kb]);
            // ---- C . S and B . C
            f32x16 G = {};
#pragma unroll
            for (int kb = 0; kb < 2 * NT; ++kb) {
                u32x4 cf[TX], bf[TX], sf[3];
                auto frag = [&](const u16 *row) { return *reinterpret_cast<const u32x4 *>(row + 16 * kb + 8 * half); };
#pragma unroll
                for (int x = 0; x < TX; ++x) cf[x] = frag(Cs[buf][x][l32]), bf[x] = frag(Bs[buf][x][l32]);
                float sv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) sv[e] = S[kb / 2][8 * (kb & 1) + e];
                split8<3, TX != 1>(sv, sf);
                product<K::IN>(G, bf, cf);     // lane = row i of C, registers = j
                product<2>(Y, sf, cf);    // lane = row i, registers = channels
            }
            // ---- M, and what it adds
            float m[16];
            const int th = (int)fresh((unsigned)(l32 - 4 * half));
            const float ci = st[1][l32], cl = st[5][l32], ei = st[4][l32];
            Y *= ei;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const Raw<float, 4> kh = load_raw<float, 4>(&st[0][8 * q + 4 * half]), kl = load_raw<float, 4>(&st[2][8 * q + 4 * half]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = G[4 * q + e] * __builtin_amdgcn_exp2f((ci - kh.v[e]) + (cl - kl.v[e]));
                    m[4 * q + e] = th >= 8 * q + e ? v : 0.0f;
                }
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                u32x4 mf[3];
                split8<3, TX != 1>(m + 8 * kb, mf);
                product<2>(Y, X[kb], mf);
            }
        }
        // ---- the state
        {
            float w[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const Raw<float, 4> u = load_raw<float, 4>(&st[3][8 * q + 4 * half]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * q + e] = u.v[e] * xc.get(4 * q + e);
            }
            if (bad < SCAN_Q) w[0] = __builtin_nanf("");
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) split8<3, TX != 1>(w + 8 * kb, W[kb]);
            const float decay = st[4][SCAN_Q - 1];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                S[nt] *= decay;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    u32x4 bf[TX];
#pragma unroll
                    for (int x = 0; x < TX; ++x) {
                        const u32x2 lo = read_columns<true>(&Bs[buf][x][0][0], NS, 16 * kb + 4 * half, 32 * nt + (l32 & 16)), hi = read_columns<true>(&Bs[buf][x][0][0], NS, 16 * kb + 8 + 4 * half, 32 * nt + (l32 & 16));
                        bf[x] = (u32x4){lo[0], lo[1], hi[0], hi[1]};
                    }
                    product<2>(S[nt], bf, W[kb]);
                }
            }
        }
        if constexpr (!STATE) {
            if (__any(bad < SCAN_Q)) {
                asm volatile("; a value that is not finite");
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (l32 >= __shfl(bad, 8 * (i / 4) + 4 * half + i % 4)) Y[i] = __builtin_nanf("");
            }
            if (g.d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const Raw<T, 4> x = load_raw<T, 4>(static_cast<const T *>(__builtin_assume_aligned(&Xs[wave][l32][8 * q + 4 * half], 4 * sizeof(T))));
#pragma unroll
                    for (int e = 0; e < 4; ++e) Y[4 * q + e] = fmaf(skip, to_f32(x.v[e]), Y[4 * q + e]);
                }
        }
        }
        if (t0 + SCAN_Q < last) {
            if (BUF == 1) __syncthreads();
            stage(BUF == 2 ? ~k & 1 : 0, t0 + SCAN_Q);
            if (k & 1) decays(t0 + SCAN_Q);
            request(t0 + 2 * SCAN_Q);
        }
        if (!STATE && works) {
            // ---- a row's channels out: register i is channel p0 + 8 (i / 4) + 4 half + i % 4
            const auto yr = rows_at(yp + (size_t)t0 * yrow, min(SCAN_Q, last - t0), yrow, width);
            const unsigned at = fresh(l32 * yrow + col);
            if (!ywide) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int c = 8 * (i / 4) + 4 * half + i % 4;
                    buffer_store(from_f32<T>(Y[i]), yr, p0 + c < P ? at + c * E : OUTSIDE);
                }
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    u32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(Y[4 * q + e]);
                    __builtin_amdgcn_raw_buffer_store_b128(v, yr, p0 + 8 * q + 4 * half < P ? at + (8 * q + 4 * half) * E : OUTSIDE, 0, 0);
                }
            } else {
                unsigned v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if constexpr (std::is_same<T, Bf16>::value) v[i] = cvt_pk_bf16(Y[2 * i], Y[2 * i + 1]);
                    else v[i] = from_f32<T>(Y[2 * i]).v | (unsigned)from_f32<T>(Y[2 * i + 1]).v << 16;
#pragma unroll
                for (int i = 0; i < 2; ++i) {   // 8 channels from 16 i + 8 half on
                    const auto a0 = __builtin_amdgcn_permlane32_swap(v[4 * i], v[4 * i + 2], false, false), a1 = __builtin_amdgcn_permlane32_swap(v[4 * i + 1], v[4 * i + 3], false, false);
                    __builtin_amdgcn_raw_buffer_store_b128((u32x4){a0[0], a1[0], a0[1], a1[1]}, yr, p0 + 16 * i + 8 * half < P ? at + (16 * i + 8 * half) * E : OUTSIDE, 0, 0);
                }
            }
        }
    }
    if (end && works) {
        const auto sr = rows_at(end + head, 1, 0, (unsigned)(P * N) * 4u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = 32 * nt + 16 * (q >> 1) + 8 * half + 4 * (q & 1);
                u32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(S[nt][4 * q + e]);
                if ((N & 3) == 0) __builtin_amdgcn_raw_buffer_store_b128(v, sr, cell(n), 0, 0);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) __builtin_amdgcn_raw_buffer_store_b32(v[e], sr, cell(n + e), 0, 0);
            }
    }
    if (STATE && works && lane == 0) cut.decays[(size_t)(slot0 + seg) * g.heads + h] = (float)total;   // several waves of a head store the same value
}

// The states from segment to segment: a thread per state value (or a few); what a segment made from zero becomes what the next one starts from.  blockIdx.y: a
// sequence, or, where there are more of them, a multiple of `rows`, for the sequence whose first one that is (one that is cut has such a row).
__global__ __launch_bounds__(256) void k_scan_carry(mdf_scan_args g, ScanSplit cut)
{
    const int b = gridDim.y == (unsigned)g.rows.B ? (int)blockIdx.y : seq_before(g.rows.row_off, g.rows.B, (int64_t)blockIdx.y * cut.rows);
    if (b < 0) return;
    const Seq s = seq_of(g.rows, b, g.state != nullptr);
    if (s.count <= cut.rows || (gridDim.y != (unsigned)g.rows.B && (s.row + cut.rows - 1) / cut.rows != (int64_t)blockIdx.y)) return;
    const int cells = g.heads * g.head_dim * g.state_dim, slot0 = (int)s.row / (cut.rows / 2), segs = (int)(((int64_t)s.count + cut.rows - 1) / cut.rows);
    for (int i = blockIdx.x * 256 + threadIdx.x; i < cells; i += gridDim.x * 256) {
        const int h = i / (g.head_dim * g.state_dim);
        float v = g.state && s.pos > 0 ? g.state[(size_t)s.slot * cells + i] : 0.0f;
        float *at = cut.states + (size_t)slot0 * cells + i;
        const float *decay = cut.decays + (size_t)slot0 * g.heads + h;
        at[0] = v;
        constexpr int AHEAD = 8;   // segments on their way from memory at once
        for (int k = 1; k < segs; k += AHEAD) {
            float own[AHEAD], d[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                const int n = min(k + e, segs - 1);
                own[e] = at[(size_t)n * cells], d[e] = decay[(size_t)(n - 1) * g.heads];
            }
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                if (k + e >= segs) break;
                v = fmaf(__builtin_amdgcn_exp2f(d[e]), v, own[e]);
                at[(size_t)(k + e) * cells] = v;
            }
        }
    }
}

// ---- one token of many sequences -----------------------------------------------------------------------------------------------------------------------
// Bound by the states' traffic, 8 bytes per state element (256 sequences of 32 x 64 x 128: 544 MB in 104 us, 5.2 TB/s); for a few sequences by latency.  A workgroup owns `rows` channels of one head: LN lanes hold a
// channel's state_dim values (V each, J times), 256 / LN channels go at once.  All its state is requested first, then the convolution of its own
// channels and of the group's B and C is made into LDS (every workgroup of a group makes B and C again: 2 N width products against a state of
// rows x N), then the state is advanced in registers and stored where it came from.
// The convolution's state is a ring: this token's entry, pos mod width, is the one entry no workgroup reads, so each input is stored by one
// workgroup at once without waiting for the others.
template <typename T, int LN, int V, int J>
__global__ __launch_bounds__(256) void k_step(mdf_step_args g, int rows)
{
    constexpr int PER = 256 / LN, MOST = 8;   // channels at once; the most a thread holds
    __shared__ float u[PER * MOST + 2 * 128];
    const int b = blockIdx.x, h = blockIdx.y, p0 = blockIdx.z * rows, r = g.heads / g.groups, grp = h / r, P = g.head_dim, N = g.state_dim, W = g.width;
    const int slot = g.slots ? g.slots[b] : b;
    if (slot < 0 || slot >= g.n_slots) {
        for (int p = threadIdx.x; g.zero_skipped && p < min(rows, P - p0); p += 256) static_cast<T *>(g.y)[(size_t)b * g.ldy + (size_t)h * P + p0 + p] = from_f32<T>(0.0f);
        return;
    }
    const unsigned pos = g.positions ? (unsigned)max(g.positions[b], 0) : 0u;
    const int channels = g.heads * P + 2 * g.groups * N, count = min(rows, P - p0);
    const int lane = threadIdx.x % LN, sub = threadIdx.x / LN;
    float *state = g.state + (((size_t)slot * g.heads + h) * P + p0) * N;
    Raw<float, V> st[MOST][J];
#pragma unroll
    for (int k = 0; k < MOST; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int p = k * PER + sub, n = (j * LN + lane) * V;
            st[k][j] = {};
            if (p < count && n < N && pos > 0) st[k][j] = load_raw<float, V>(state + (size_t)p * N + n);
        }
    T *ring = static_cast<T *>(g.conv_state) + (size_t)slot * W * channels;
    for (int i = threadIdx.x; i < count + 2 * N; i += 256) {
        const int c = i < count ? h * P + p0 + i : g.heads * P + (i < count + N ? grp * N + i - count : (g.groups + grp) * N + i - count - N);
        const T now = static_cast<const T *>(g.xbc)[(size_t)b * g.ldx + c];
        float v = g.conv_bias ? g.conv_bias[c] : 0.0f;
#pragma unroll 4
        for (unsigned back = W - 1; back > 0; --back)
            if (pos >= back) v = fmaf(g.conv_weight[(size_t)(W - 1 - back) * channels + c], to_f32(ring[(size_t)((pos - back) % W) * channels + c]), v);
        v = fmaf(g.conv_weight[(size_t)(W - 1) * channels + c], to_f32(now), v);
        u[i < count ? i : i - count + PER * MOST] = silu(v);
        if (i < count || (h % r == 0 && p0 == 0)) ring[(size_t)(pos % W) * channels + c] = now;
    }
    const float delta = softplus(load_any(g.dt, (size_t)b * g.lddt + h, g.dt_dtype) + (g.dt_bias ? g.dt_bias[h] : 0.0f)), decay = expf(delta * g.a[h]);
    const float skip = g.d ? g.d[h] : 0.0f;
    __syncthreads();
    float B[J][V], C[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int n = (j * LN + lane) * V + i;
            B[j][i] = n < N ? u[PER * MOST + n] : 0.0f;
            C[j][i] = n < N ? u[PER * MOST + N + n] : 0.0f;
        }
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
        const int p = k * PER + sub;
        if (k * PER >= count) break;
        const float x = p < count ? u[p] : 0.0f, dx = delta * x;
        float y = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int n = (j * LN + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                st[k][j].v[i] = fmaf(decay, st[k][j].v[i], dx * B[j][i]);
                y = fmaf(st[k][j].v[i], C[j][i], y);
            }
            if (p < count && n < N) store_raw(state + (size_t)p * N + n, st[k][j]);
        }
#pragma unroll
        for (int m = 1; m < LN; m <<= 1) y += __shfl_xor(y, m);
        if (lane == 0 && p < count) static_cast<T *>(g.y)[(size_t)b * g.ldy + (size_t)h * P + p0 + p] = from_f32<T>(g.d ? fmaf(skip, x, y) : y);
    }
}

// ---- block norms ------------------------------------------------------------------------------------------------------------------------------------
// One pass: a row's inputs are requested together, live in registers as f32 through both norms and leave once.  TPR threads per (row, group) hold
// VPT x 8 values each; TPR = 64 are four rows per workgroup, whose sums need no LDS.  Bound by memory: 65 536 rows of 2 048 with a gate in bfloat16 (805 MB) take
// 150 us, 5.4 TB/s.  Sums: in order over a thread's values, then a tree over lanes -- the same for every row, whatever the batch.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *part)
{
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += part[i];
    }
    return v;
}

// v / d for many v at two instructions each: the reciprocal and what it is off by, so the quotient is rounded once (a lone reciprocal rounds twice)
struct Reciprocal {
    float q, rest;
    __device__ __forceinline__ explicit Reciprocal(float d) : q(1.0f / d), rest(d < __builtin_inff() ? fmaf(-d, q, 1.0f) * q : 0.0f) {}
    __device__ __forceinline__ float times(float v) const { return fmaf(v, q, v * rest); }
};

// thread t of a row holds the 8 values from (v TPR + t) 8 on; a row's last few are taken one by one
template <typename T, typename R, int TPR, int VPT>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void k_block_norm(mdf_block_norm_args g)
{
    __shared__ float part[16];
    const int t = threadIdx.x % TPR, width = g.dim / g.groups, c0 = blockIdx.y * width;
    const size_t row = TPR == 64 ? (size_t)blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x;
    if (row >= (size_t)g.rows) return;    // whole waves (TPR = 64) only
    const T *s = static_cast<const T *>(g.s) + row * g.lds + c0, *gate = static_cast<const T *>(g.gate) + row * g.ldg + c0;
    const R *res = static_cast<const R *>(g.residual) + row * g.ldr + c0;
    auto left = [&](int v) { return width - (v * TPR + t) * 8; };   // values from vector v's first to the row's end
    auto load = [&](auto *p, auto &raw, int v) {
        const int n = left(v);
        p += (v * TPR + t) * 8;
        raw = {};
        if (n >= 8) raw = load_raw<typename std::remove_const<typename std::remove_pointer<decltype(p)>::type>::type, 8>(p);
        else if (n > 0)
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < n) raw.v[e] = p[e];
    };
    auto param = [&](const float *p, int v) {   // 8 parameters of vector v
        Raw<float, 8> r;
        load(p + c0, r, v);
        return r;
    };
    Raw<T, 8> rs[VPT], rg[VPT];
    Raw<R, 8> rr[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) load(s, rs[v], v);
    if (g.gate)
#pragma unroll
        for (int v = 0; v < VPT; ++v) load(gate, rg[v], v);
    if (g.residual)
#pragma unroll
        for (int v = 0; v < VPT; ++v) load(res, rr[v], v);
    float x[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[v][e] = to_f32(rs[v].v[e]);
    auto gated = [&]() {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float z = to_f32(rg[v].v[e]);
                x[v][e] *= g.gate_act == MDF_ACT_SILU ? silu(z) : g.gate_act == MDF_ACT_SIGMOID ? sigmoid(z) : z;
            }
        }
    };
    // values beyond the row are zeros going in; the centred sum of squares leaves them out again
    auto norm = [&](const float *weight, const float *bias) {
        float mean = 0.0f, sum = 0.0f;
        if (g.center) {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) mean += x[v][e];
            mean = row_sum<TPR>(mean, part) / (float)width;
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (e < left(v)) x[v][e] -= mean;
                sum = fmaf(x[v][e], x[v][e], sum);
            }
        const Reciprocal q(sqrtf(row_sum<TPR>(sum, part) / (float)width + g.eps));
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            Raw<float, 8> w = param(weight, v), o = {};
            if (bias) o = param(bias, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[v][e] = fmaf(q.times(x[v][e]), w.v[e], o.v[e]);
        }
    };
    auto store = [&](auto *p) {
        typedef typename std::remove_pointer<decltype(p)>::type O;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int n = left(v);
            O *q = p + (v * TPR + t) * 8;
            if (n >= 8) store_f32<O, 8>(q, x[v]);
            else if (n > 0)
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (e < n) q[e] = from_f32<O>(x[v][e]);
        }
    };
    if (g.gate && g.gate_first) gated();
    if (g.post_weight) norm(g.post_weight, g.post_bias);
    if (g.gate && !g.gate_first) gated();
    if (g.residual) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            Raw<float, 8> k = {};
            if (g.scale_vec) k = param(g.scale_vec, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[v][e] = fmaf(g.scale_vec ? g.scale * k.v[e] : g.scale, x[v][e], to_f32(rr[v].v[e]));
        }
        store(static_cast<R *>(g.residual_out) + row * g.ldro + c0);
    }
    if (g.pre_weight) norm(g.pre_weight, g.pre_bias);
    if (g.out) store(static_cast<T *>(g.out) + row * g.ldo + c0);
}

// Rows wider than the registers of 1 024 threads hold (16 384 values): one workgroup walks the row three times, the second and third out of L2
__device__ __forceinline__ float block_sum(float v)
{
    __shared__ float part[4];
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}
template <typename T, typename R>
__global__ __launch_bounds__(256) void k_block_norm_walk(mdf_block_norm_args g)
{
    const size_t row = blockIdx.x;
    const int width = g.dim / g.groups, c0 = blockIdx.y * width, c1 = c0 + width;
    const T *s = static_cast<const T *>(g.s) + row * g.lds, *gate = g.gate ? static_cast<const T *>(g.gate) + row * g.ldg : nullptr;
    const R *res = g.residual ? static_cast<const R *>(g.residual) + row * g.ldr : nullptr;
    auto gated = [&](int c) {
        const float z = to_f32(gate[c]);
        return g.gate_act == MDF_ACT_SILU ? silu(z) : g.gate_act == MDF_ACT_SIGMOID ? sigmoid(z) : z;
    };
    auto first = [&](int c) { return to_f32(s[c]) * (gate && g.gate_first ? gated(c) : 1.0f); };
    float m1 = 0.0f, m2 = 0.0f, sum = 0.0f;
    Reciprocal q1(1.0f), q2(1.0f);
    if (g.post_weight) {
        if (g.center) {
            for (int c = c0 + threadIdx.x; c < c1; c += 256) sum += first(c);
            m1 = block_sum(sum) / width;
        }
        sum = 0.0f;
        for (int c = c0 + threadIdx.x; c < c1; c += 256) sum += (first(c) - m1) * (first(c) - m1);
        q1 = Reciprocal(sqrtf(block_sum(sum) / width + g.eps));
    }
    auto after = [&](int c) {
        float v = first(c);
        if (g.post_weight) v = q1.times(v - m1) * g.post_weight[c] + (g.post_bias ? g.post_bias[c] : 0.0f);
        if (gate && !g.gate_first) v *= gated(c);
        return res ? to_f32(res[c]) + g.scale * (g.scale_vec ? g.scale_vec[c] : 1.0f) * v : v;
    };
    if (g.pre_weight) {
        sum = 0.0f;
        if (g.center) {
            for (int c = c0 + threadIdx.x; c < c1; c += 256) sum += after(c);
            m2 = block_sum(sum) / width;
        }
        sum = 0.0f;
        for (int c = c0 + threadIdx.x; c < c1; c += 256) sum += (after(c) - m2) * (after(c) - m2);
        q2 = Reciprocal(sqrtf(block_sum(sum) / width + g.eps));
    }
    for (int c = c0 + threadIdx.x; c < c1; c += 256) {
        const float v = after(c);
        if (res) static_cast<R *>(g.residual_out)[row * g.ldro + c] = from_f32<R>(v);
        if (g.pre_weight) static_cast<T *>(g.out)[row * g.ldo + c] = from_f32<T>(q2.times(v - m2) * g.pre_weight[c] + (g.pre_bias ? g.pre_bias[c] : 0.0f));
        else if (!res) static_cast<T *>(g.out)[row * g.ldo + c] = from_f32<T>(v);
    }
}

// ---- argument checks -------------------------------------------------------------------------------------------------------------------------
static size_t dt_size(int dt) { return dt == MDF_DT_F32 ? 4 : dt == MDF_DT_BF16 || dt == MDF_DT_F16 ? 2 : 0; }

// Whether two arrays of `rows` rows share a byte: row starts `ld` elements apart, `width` elements used of each.  Column ranges of one wider
// array (equal strides) do not overlap where the columns do not.
static bool overlap(const void *p, int64_t ldp, int64_t wp, size_t ep, const void *q, int64_t ldq, int64_t wq, size_t eq, int64_t rows)
{
    if (!p || !q || rows <= 0 || wp <= 0 || wq <= 0) return false;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    const uintptr_t ae = a + ((uintptr_t)(rows - 1) * ldp + wp) * ep, be = b + ((uintptr_t)(rows - 1) * ldq + wq) * eq;
    if (ae <= b || be <= a) return false;
    const uintptr_t la = (uintptr_t)ldp * ep, lb = (uintptr_t)ldq * eq;
    if (la == lb && la > 0 && rows > 1) {
        const uintptr_t d = b >= a ? (b - a) % la : (la - (a - b) % la) % la;   // where q's columns begin in p's rows
        if (d >= wp * ep && d + wq * eq <= la) return false;
    }
    return true;
}

template <typename T, typename R, int TPR, int VPT>
static void norm_launch(const mdf_block_norm_args &a, hipStream_t st)
{
    const dim3 grid((unsigned)(TPR == 64 ? (a.rows + 3) / 4 : a.rows), a.groups), block(TPR == 64 ? 256 : TPR);
    hipLaunchKernelGGL((k_block_norm<T, R, TPR, VPT>), grid, block, 0, st, a);
}
// As few threads as hold the row in one vector each, to 512 of them; then two vectors.  128 Mi bfloat16 values in rows of `width` with a gate, us:
//   512: 64 threads x 1 vector 145-158, 128 x 1 231-246        1 024: 128 x 1 144, 64 x 2 166, 256 x 1 233       2 048: 256 x 1 143, 128 x 2 160, 64 x 4 311, 512 x 1 255
//   4 096: 512 x 1 152, 256 x 2 188, 1 024 x 1 383             8 192: 512 x 2 200, 1 024 x 1 228, 256 x 4 301    16 384: 1 024 x 2 215, the walk 500
template <typename T, typename R>
static void norm_by_width(const mdf_block_norm_args &a, hipStream_t st)
{
    const int width = a.dim / a.groups;
    if (width <= 512) norm_launch<T, R, 64, 1>(a, st);
    else if (width <= 1024) norm_launch<T, R, 128, 1>(a, st);
    else if (width <= 2048) norm_launch<T, R, 256, 1>(a, st);
    else if (width <= 4096) norm_launch<T, R, 512, 1>(a, st);
    else if (width <= 8192) norm_launch<T, R, 512, 2>(a, st);
    else if (width <= 16384) norm_launch<T, R, 1024, 2>(a, st);
    else hipLaunchKernelGGL((k_block_norm_walk<T, R>), dim3((unsigned)a.rows, a.groups), dim3(256), 0, st, a);
}

// How a call's sequences are cut.  Unsplit there is a workgroup per sequence and four blocks of 32 channels.
struct ScanPlan {
    int unit_blocks, seg_rows, slots, items;
    size_t state_floats, decay_floats;
};
static ScanPlan scan_plan(const mdf_scan_args &a)
{
    ScanPlan p = {};
    const int pblocks = (a.head_dim + 31) / 32;
    p.unit_blocks = a.groups * ((a.heads / a.groups * pblocks + SCAN_WAVES - 1) / SCAN_WAVES);
    // `even`: rows per workgroup if all were equally long, two per CU (512).  A sequence much longer than that is what a call waits for, and the calls it
    // holds up are cut although making the states first costs half as much again: 32 768 rows of 16 heads take 162 us in 64 segments (191 in 128, 182
    // in 32, 580 in 8); 48 mixed lengths to 1 024 of 8 heads in float32 127 us in segments of 256, 150 uncut.  Under 256 rows the carried states outweigh it.
    // Beside 32 / 128 sequences of one row the 32 768 rows take 187 / 207 us, 3 000 where they are not cut.
    const int64_t even = a.rows.R * p.unit_blocks / 512;
    if (a.rows.max_len > 512 && (int64_t)a.rows.max_len * 2 > even * 5) {
        const int rows = (int)std::max<int64_t>(256, (even + 63) / 64 * 64);
        if (a.rows.max_len > rows) {
            // some 1 024 / unit_blocks slots at most, since rows >= even: a workspace of 65 MiB whatever the lengths, for a workgroup's part of a state is 128 x 128
            p.seg_rows = rows;
            p.slots = (int)(a.rows.R * 2 / rows);
            p.state_floats = (size_t)p.slots * a.heads * a.head_dim * a.state_dim;
            p.decay_floats = (size_t)p.slots * a.heads;
        }
    }
    p.items = a.rows.B + p.slots;
    return p;
}

template <typename T, int NT, bool WORDS>
static void scan_launch(const mdf_scan_args &a, const ScanPlan &p, void *workspace, hipStream_t st)
{
    ScanSplit cut = {p.seg_rows, p.slots, static_cast<float *>(workspace), static_cast<float *>(workspace) + p.state_floats};
    const int items = p.items;
    const unsigned blocks = (unsigned)((items + 7) / 8 * 8) * p.unit_blocks;
    const dim3 grid(std::min(blocks, GRID_X), (blocks + GRID_X - 1) / GRID_X), block(64 * SCAN_WAVES);
    if (p.seg_rows) {
        hipLaunchKernelGGL((k_scan<T, NT, true, WORDS>), grid, block, 0, st, a, cut, items, p.unit_blocks);
        // some 4 096 workgroups: most find no sequence where the few long ones are among many
        const unsigned y = (unsigned)std::min<int64_t>(a.rows.B, a.rows.R / p.seg_rows + 1), x = (unsigned)((a.heads * a.head_dim * a.state_dim + 255) / 256);
        hipLaunchKernelGGL(k_scan_carry, dim3(y == 1 ? x : std::min(x, std::max(4096 / y, 1u)), y), dim3(256), 0, st, a, cut);
    }
    hipLaunchKernelGGL((k_scan<T, NT, false, WORDS>), grid, block, 0, st, a, cut, items, p.unit_blocks);
}
template <typename T, bool WORDS>
static void scan_by_state(const mdf_scan_args &a, const ScanPlan &p, void *workspace, hipStream_t st)
{
    switch ((a.state_dim + 31) / 32) {
    case 1: scan_launch<T, 1, WORDS>(a, p, workspace, st); break;
    case 2: scan_launch<T, 2, WORDS>(a, p, workspace, st); break;
    case 3: scan_launch<T, 3, WORDS>(a, p, workspace, st); break;
    default: scan_launch<T, 4, WORDS>(a, p, workspace, st); break;
    }
}
template <typename T>
static void scan_by_alignment(const mdf_scan_args &a, const ScanPlan &p, void *workspace, hipStream_t st)
{
    if constexpr (sizeof(T) == 2) {
        const bool words = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.b) | reinterpret_cast<uintptr_t>(a.c)) & 3) == 0 && ((a.ldx | a.ldb | a.ldc) & 1) == 0 &&
                           (a.heads == 1 || a.head_dim % 2 == 0) && (a.groups == 1 || a.state_dim % 2 == 0);
        if (!words) return scan_by_state<T, false>(a, p, workspace, st);
    }
    scan_by_state<T, true>(a, p, workspace, st);
}

template <typename T>
static void step_launch(const mdf_step_args &a, hipStream_t st)
{
    const int N = a.state_dim;
    const bool wide = N % 4 == 0;   // else one value at a time
    const int ln = wide ? (N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32) : N <= 16 ? 16 : N <= 32 ? 32 : 64;
    const int per = 256 / ln;
    // Channels per workgroup: as many as a thread's registers hold (8 x `per`) while that leaves two workgroups per CU, fewer for few sequences: each workgroup makes
    // B and C again.  32 heads of 64 channels x 128, us with 8 / 16 / 32 / 64 channels: 2 sequences 4.9 / 4.9 / 5.5 / 6.5, 4: 6.3 / 5.4 / 5.8 / 6.8,
    // 8: 10.1 / 7.2 / 6.4 / 7.3, 16: 15.8 / 11.1 / 8.8 / 8.3, 128: 95 / 59 / 51 / 45.
    int rows = std::min(a.head_dim, 8 * per);
    while (rows > per && (int64_t)a.B * a.heads * ((a.head_dim + rows - 1) / rows) < 512) rows = std::max(per, (rows / 2 + per - 1) / per * per);
    const dim3 grid((unsigned)a.B, a.heads, (a.head_dim + rows - 1) / rows);
#define MDF_S(ln_, v_, j_) hipLaunchKernelGGL((k_step<T, ln_, v_, j_>), grid, dim3(256), 0, st, a, rows)
    if (wide) {
        if (ln == 4) MDF_S(4, 4, 1);
        else if (ln == 8) MDF_S(8, 4, 1);
        else if (ln == 16) MDF_S(16, 4, 1);
        else MDF_S(32, 4, 1);
    } else {
        if (ln == 16) MDF_S(16, 1, 1);
        else if (ln == 32) MDF_S(32, 1, 1);
        else MDF_S(64, 1, 2);
    }
#undef MDF_S
}

template <typename T, int V>
static void conv_launch(const mdf_conv_args &a, int steps, int lanes, dim3 grid, hipStream_t st)
{
    switch (a.width) {
#define MDF_W(w_) case w_: hipLaunchKernelGGL((k_conv<T, V, w_>), grid, dim3(256), 0, st, a, steps, lanes); break;
        MDF_W(1) MDF_W(2) MDF_W(3) MDF_W(4) MDF_W(5) MDF_W(6) MDF_W(7) MDF_W(8)
#undef MDF_W
    }
}

static int check_rows(const mdf_seq_rows &r, const char *who, bool kept)
{
    MDF_REQUIRE(r.B >= 0 && r.R >= 0 && r.R < (int64_t)1 << 31, "%s: B=%d sequences, R=%lld rows", who, r.B, (long long)r.R);
    MDF_REQUIRE(r.B == 0 || (r.lengths && r.row_off), "%s: lengths or row_off is NULL", who);
    MDF_REQUIRE(r.max_len >= 0 && r.max_len <= r.R, "%s: max_len=%d of %lld rows", who, r.max_len, (long long)r.R);
    if (kept) MDF_REQUIRE(r.n_slots >= 0 && (r.slots || r.n_slots >= r.B), "%s: %d states for %d sequences without slots", who, r.n_slots, r.B);
    return MDF_OK;
}

}  // namespace mdf

using namespace mdf;

#define MDF_BY_TYPE(dt_, T_, ...)                                                              \
    do {                                                                                       \
        if ((dt_) == MDF_DT_F32) { typedef float T_; __VA_ARGS__; }                            \
        else if ((dt_) == MDF_DT_BF16) { typedef ::mdf::Bf16 T_; __VA_ARGS__; }                \
        else { typedef ::mdf::F16 T_; __VA_ARGS__; }                                           \
    } while (0)

extern "C" {

int mdf_causal_conv_dev(const mdf_conv_args *a, void *stream)
{
    MDF_REQUIRE(a, "causal_conv_dev: NULL argument");
    if (int rc = check_rows(a->rows, "causal_conv_dev", a->state != nullptr)) return rc;
    MDF_REQUIRE(dt_size(a->dtype), "causal_conv_dev: dtype %d is not f32, bf16 or f16", a->dtype);
    MDF_REQUIRE(a->channels > 0 && a->width >= 1 && a->width <= 8, "causal_conv_dev: channels=%d, width=%d (1..8)", a->channels, a->width);
    if (a->rows.B == 0 || a->rows.R == 0) return MDF_OK;
    MDF_REQUIRE(a->x && a->weight && a->out, "causal_conv_dev: NULL argument");
    MDF_REQUIRE(a->ldx >= 0 && (a->ldo >= a->channels || a->rows.R == 1), "causal_conv_dev: row strides %lld, %lld for %d channels", (long long)a->ldx, (long long)a->ldo, a->channels);
    const size_t e = dt_size(a->dtype);
    MDF_REQUIRE(!overlap(a->x, a->ldx, a->channels, e, a->out, a->ldo, a->channels, e, a->rows.R), "causal_conv_dev: out overlaps x");
    const int v = a->channels >= 16 / (int)e ? 16 / (int)e : 1;
    const int lanes = (a->channels + v - 1) / v;
    // Tiles per thread: further ones save the weights, the rows in front and a search, and cost parallel threads; they pay once one tile each is more than
    // the waves that are resident at once.  1 / 2 / 4 tiles, us (640 channels; threads of one tile in units of 65 536, one wave per SIMD):
    //   bf16  1.7 units: width 4 15.0 / 16.8 / 21.3, 8 22.8 / 28.1 / 34.7      3.3: width 2 16.9 / 17.8 / 18.1, 4 23.3 / 21.1 / 21.9, 8 38.6 / 29.2 / 30.3
    //         5.3: width 4 30.6 / 26.3 / 28.6, 5 37.1 / 32.5 / 30.8            21: width 2 71.8 / 73.2 / 78.6, 4 101 / 84.5 / 84.8, 8 169 / 138 / 111
    //   f32   3.3: width 4 15.3 / 15.8 / 16.7                                  6.6: width 2 21.1 / 20.4 / 19.8, 4 24.0 / 22.7 / 21.6, 8 41.3 / 35.0 / 27.0
    const int64_t tiles = (a->rows.R + CONV_ROWS - 1) / CONV_ROWS, units = tiles * lanes / 65536;
    int steps = 1;
    if (e == 4) steps = units >= 6 ? 4 : 1;
    else if (a->width > 2 && units >= 3) steps = a->width > 4 && units >= 5 ? 4 : 2;
    const int64_t threads = (tiles + steps - 1) / steps * lanes;
    MDF_REQUIRE((threads + 255) / 256 < 2 * (int64_t)GRID_X, "causal_conv_dev: %lld rows of %d channels are too many", (long long)a->rows.R, a->channels);
    if (int rc = require_device()) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)((threads + 255) / 256));
    MDF_BY_TYPE(a->dtype, T, {
        if (v > 1) conv_launch<T, 16 / sizeof(T)>(*a, steps, lanes, grid, st);
        else conv_launch<T, 1>(*a, steps, lanes, grid, st);
    });
    MDF_HIP(hipGetLastError());
    return MDF_OK;
}

// Every argument of the scan that does not take the device to check.
static int check_scan(const mdf_scan_args *a)
{
    MDF_REQUIRE(a, "selective_scan_dev: NULL argument");
    if (int rc = check_rows(a->rows, "selective_scan_dev", a->state != nullptr)) return rc;
    MDF_REQUIRE(dt_size(a->dtype) && dt_size(a->dt_dtype), "selective_scan_dev: dtype %d / %d is not f32, bf16 or f16", a->dtype, a->dt_dtype);
    MDF_REQUIRE(a->heads > 0 && a->heads <= 65535 && a->groups > 0 && a->heads % a->groups == 0, "selective_scan_dev: %d heads in %d groups", a->heads, a->groups);
    MDF_REQUIRE(a->head_dim >= 1 && a->head_dim <= 256 && a->state_dim >= 1 && a->state_dim <= 128, "selective_scan_dev: head_dim=%d (1..256), state_dim=%d (1..128)",
                a->head_dim, a->state_dim);
    if (a->rows.B == 0 || a->rows.R == 0) return MDF_OK;
    MDF_REQUIRE(a->x && a->b && a->c && a->dt && a->y, "selective_scan_dev: NULL argument");
    MDF_REQUIRE(a->a, "selective_scan_dev: a is NULL");
    const int64_t R = a->rows.R, hp = (int64_t)a->heads * a->head_dim, gn = (int64_t)a->groups * a->state_dim;
    MDF_REQUIRE(R == 1 || (a->ldx >= hp && a->ldb >= gn && a->ldc >= gn && a->lddt >= a->heads && a->ldy >= hp), "selective_scan_dev: a row stride is below its row's width");
    // a chunk of 32 rows is addressed with 32-bit byte offsets
    MDF_REQUIRE(a->ldx < (int64_t)1 << 23 && a->ldb < (int64_t)1 << 23 && a->ldc < (int64_t)1 << 23 && a->ldy < (int64_t)1 << 23 && hp < (int64_t)1 << 23 && gn < (int64_t)1 << 23,
                "selective_scan_dev: a row or its stride of 2^23 values or more");
    const size_t e = dt_size(a->dtype);
    MDF_REQUIRE(!overlap(a->x, a->ldx, hp, e, a->y, a->ldy, hp, e, R) && !overlap(a->b, a->ldb, gn, e, a->y, a->ldy, hp, e, R) &&
                    !overlap(a->c, a->ldc, gn, e, a->y, a->ldy, hp, e, R) && !overlap(a->dt, a->lddt, a->heads, dt_size(a->dt_dtype), a->y, a->ldy, hp, e, R),
                "selective_scan_dev: y overlaps an input");
    const ScanPlan p = scan_plan(*a);
    MDF_REQUIRE(((int64_t)p.items + 7) / 8 * 8 * p.unit_blocks < (int64_t)1 << 31 && (int64_t)a->heads * a->head_dim * a->state_dim < (int64_t)1 << 31,
                "selective_scan_dev: %d sequences of %d heads are too many for one call", a->rows.B, a->heads);
    return MDF_OK;
}

size_t mdf_scan_workspace_bytes(const mdf_scan_args *a)
{
    if (!a || a->rows.B <= 0 || a->rows.R <= 0 || check_scan(a) != MDF_OK) return 0;
    const ScanPlan p = scan_plan(*a);
    return (p.state_floats + p.decay_floats) * sizeof(float);
}

int mdf_selective_scan_dev(const mdf_scan_args *a, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_scan(a)) return rc;
    if (a->rows.B == 0 || a->rows.R == 0) return MDF_OK;
    mdf_scan_args one = *a;
    if (a->rows.R == 1) one.ldx = one.ldy = ((int64_t)a->heads * a->head_dim + 1) & ~1ll, one.ldb = one.ldc = ((int64_t)a->groups * a->state_dim + 1) & ~1ll, a = &one;   // the strides of a single row say nothing
    const ScanPlan p = scan_plan(*a);
    const size_t need = (p.state_floats + p.decay_floats) * sizeof(float);
    if (need > workspace_bytes || (need && !workspace))
        return fail(MDF_ECAPACITY, "selective_scan_dev: workspace of %zu bytes is smaller than %zu", workspace ? workspace_bytes : 0, need);
    if (int rc = require_device()) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    MDF_BY_TYPE(a->dtype, T, scan_by_alignment<T>(*a, p, workspace, st));
    MDF_HIP(hipGetLastError());
    return MDF_OK;
}

int mdf_selective_step_dev(const mdf_step_args *a, void *stream)
{
    MDF_REQUIRE(a, "selective_step_dev: NULL argument");
    MDF_REQUIRE(dt_size(a->dtype) && dt_size(a->dt_dtype), "selective_step_dev: dtype %d / %d is not f32, bf16 or f16", a->dtype, a->dt_dtype);
    MDF_REQUIRE(a->heads > 0 && a->heads <= 65535 && a->groups > 0 && a->heads % a->groups == 0, "selective_step_dev: %d heads in %d groups", a->heads, a->groups);
    MDF_REQUIRE(a->head_dim >= 1 && a->head_dim <= 256 && a->state_dim >= 1 && a->state_dim <= 128, "selective_step_dev: head_dim=%d (1..256), state_dim=%d (1..128)",
                a->head_dim, a->state_dim);
    MDF_REQUIRE(a->width >= 1 && a->width <= 8, "selective_step_dev: width=%d (1..8)", a->width);
    MDF_REQUIRE(a->B >= 0 && a->n_slots >= 0 && (a->slots || a->n_slots >= a->B), "selective_step_dev: %d states for %d sequences without slots", a->n_slots, a->B);
    if (a->B == 0) return MDF_OK;
    MDF_REQUIRE(a->xbc && a->dt && a->conv_weight && a->a && a->conv_state && a->state && a->y, "selective_step_dev: NULL argument");
    const int64_t hp = (int64_t)a->heads * a->head_dim, ch = hp + 2 * (int64_t)a->groups * a->state_dim;
    MDF_REQUIRE(ch < (int64_t)1 << 31, "selective_step_dev: %lld channels", (long long)ch);
    MDF_REQUIRE(a->ldx >= 0 && a->lddt >= 0 && (a->ldy >= hp || a->B == 1), "selective_step_dev: a row stride is negative or y's is below %lld", (long long)hp);
    const size_t e = dt_size(a->dtype);
    MDF_REQUIRE(!overlap(a->xbc, a->ldx, ch, e, a->y, a->ldy, hp, e, a->B) && !overlap(a->dt, a->lddt, a->heads, dt_size(a->dt_dtype), a->y, a->ldy, hp, e, a->B),
                "selective_step_dev: y overlaps an input");
    if (int rc = require_device()) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    mdf_step_args k = *a;
    for (int64_t b = 0; b < a->B; b += GRID_X) {   // a workgroup at least per sequence, in x
        k.B = (int32_t)std::min<int64_t>(GRID_X, a->B - b);
        k.xbc = static_cast<const char *>(a->xbc) + (size_t)b * a->ldx * e;
        k.dt = static_cast<const char *>(a->dt) + (size_t)b * a->lddt * dt_size(a->dt_dtype);
        k.y = static_cast<char *>(a->y) + (size_t)b * a->ldy * e;
        if (a->positions) k.positions = a->positions + b;
        if (a->slots) k.slots = a->slots + b;
        else {
            k.n_slots = a->n_slots - (int32_t)b;
            k.conv_state = static_cast<char *>(a->conv_state) + (size_t)b * a->width * ch * e;
            k.state = a->state + (size_t)b * hp * a->state_dim;
        }
        MDF_BY_TYPE(a->dtype, T, step_launch<T>(k, st));
    }
    MDF_HIP(hipGetLastError());
    return MDF_OK;
}

int mdf_block_norm_dev(const mdf_block_norm_args *a, void *stream)
{
    MDF_REQUIRE(a, "block_norm_dev: NULL argument");
    const size_t e = dt_size(a->dtype), er = a->residual ? dt_size(a->residual_dtype) : 0;
    MDF_REQUIRE(e, "block_norm_dev: dtype %d is not f32, bf16 or f16", a->dtype);
    MDF_REQUIRE(!a->residual || a->residual_dtype == MDF_DT_F32 || a->residual_dtype == a->dtype, "block_norm_dev: residual of type %d beside %d", a->residual_dtype, a->dtype);
    MDF_REQUIRE(a->rows >= 0 && a->rows < (int64_t)1 << 31 && a->dim >= 1 && a->dim <= 32768, "block_norm_dev: rows=%lld, dim=%d (1..32768)", (long long)a->rows, a->dim);
    MDF_REQUIRE(a->groups >= 1 && a->groups <= 65535 && a->dim % a->groups == 0, "block_norm_dev: dim=%d in %d groups", a->dim, a->groups);
    MDF_REQUIRE(a->groups == 1 || !a->pre_weight, "block_norm_dev: groups=%d with a pre-norm", a->groups);
    MDF_REQUIRE(a->gate_act >= MDF_ACT_NONE && a->gate_act <= MDF_ACT_SIGMOID, "block_norm_dev: gate_act=%d", a->gate_act);
    MDF_REQUIRE(a->post_weight || !a->post_bias, "block_norm_dev: post_bias without post_weight");
    MDF_REQUIRE(a->pre_weight || !a->pre_bias, "block_norm_dev: pre_bias without pre_weight");
    MDF_REQUIRE(a->residual || !a->scale_vec, "block_norm_dev: scale_vec without a residual");
    if (a->rows == 0) return MDF_OK;
    const bool has_out = a->pre_weight || !a->residual;
    MDF_REQUIRE(a->s && (!a->residual || a->residual_out) && (!has_out || a->out), "block_norm_dev: NULL argument");
    const int64_t d = a->dim;
    MDF_REQUIRE(a->lds >= 0 && a->ldg >= 0 && a->ldr >= 0 && (a->rows == 1 || ((!a->residual || a->ldro >= d) && (!has_out || a->ldo >= d))),
                "block_norm_dev: a row stride is negative or an output's is below %d", a->dim);
    struct { const void *p; int64_t ld; size_t e; } in[3] = {{a->s, a->lds, e}, {a->gate, a->ldg, e}, {a->residual, a->ldr, er}},
                                                  out[2] = {{a->residual ? a->residual_out : nullptr, a->ldro, er}, {has_out ? a->out : nullptr, a->ldo, e}};
    for (auto &o : out)
        for (auto &i : in) {
            const bool same = o.p == i.p && o.e == i.e && (o.ld == i.ld || a->rows == 1);
            MDF_REQUIRE(same || !overlap(i.p, i.ld, d, i.e, o.p, o.ld, d, o.e, a->rows), "block_norm_dev: an output overlaps an input without being it");
        }
    MDF_REQUIRE(!overlap(out[0].p, out[0].ld, d, er, out[1].p, out[1].ld, d, e, a->rows), "block_norm_dev: the outputs overlap");
    if (int rc = require_device()) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    mdf_block_norm_args k = *a;
    constexpr int64_t ROWS = 1 << 21;   // of one launch: up to 1 024 threads each in x
    for (int64_t r = 0; r < a->rows; r += ROWS) {
        auto at = [&](auto *p, int64_t ld, size_t size) { return p ? (decltype(p))((uintptr_t)p + (size_t)r * ld * size) : p; };
        k.rows = std::min(ROWS, a->rows - r);
        k.s = at(a->s, a->lds, e), k.gate = at(a->gate, a->ldg, e), k.residual = at(a->residual, a->ldr, er);
        k.residual_out = at(a->residual_out, a->ldro, er), k.out = has_out ? at(a->out, a->ldo, e) : nullptr;
        MDF_BY_TYPE(a->dtype, T, {
            if (a->residual && a->residual_dtype == MDF_DT_F32) norm_by_width<T, float>(k, st);
            else norm_by_width<T, T>(k, st);
        });
    }
    MDF_HIP(hipGetLastError());
    return MDF_OK;
}

}  // extern "C"
