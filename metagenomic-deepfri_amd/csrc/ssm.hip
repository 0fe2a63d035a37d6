// ssm.hip -- operators of a state-space language-model block over packed residue rows: short causal convolution, selective scan, both for one
// token, and the norms around the block (include/mdfri.h "Operators of a state-space language-model block").
#include "common.h"

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

__device__ __forceinline__ float silu(float v) { return v / (1.0f + __expf(-v)); }
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + __expf(-v)); }
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))); }
// one value of any of the three types, by code (uniform): the step sizes dt, which are read once per head and row
__device__ __forceinline__ float load_any(const void *p, size_t i, int dt)
{
    return dt == MDF_DT_F32 ? static_cast<const float *>(p)[i] : dt == MDF_DT_BF16 ? to_f32(static_cast<const Bf16 *>(p)[i]) : to_f32(static_cast<const F16 *>(p)[i]);
}

// What a kernel knows of a sequence; count < 0: skipped (its slot is outside the pool, or it has no rows)
struct Seq {
    int64_t row;      // first row
    int count;        // rows
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
    s.count = (int)n;
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

// ---- the short causal convolution: simple form, one thread per row and channel ----------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_conv_simple(mdf_conv_args g)
{
    const int64_t row = blockIdx.x;
    const int b = seq_before(g.rows.row_off, g.rows.B, row);
    if (b < 0) return;
    const Seq s = seq_of(g.rows, b, g.state != nullptr);
    const int64_t t = row - s.row;
    if (t >= s.count) return;
    const T *x = static_cast<const T *>(g.x);
    const T *ring = static_cast<const T *>(g.state) + (size_t)s.slot * g.width * g.channels;
    for (int c = threadIdx.x; c < g.channels; c += 256) {
        float v = g.bias ? g.bias[c] : 0.0f;
        for (int k = 0; k < g.width; ++k) {
            const int back = g.width - 1 - k;
            float u = 0.0f;
            if (t >= back) u = to_f32(x[(size_t)(row - back) * g.ldx + c]);
            else if (g.state && s.pos + t >= back) u = to_f32(ring[(size_t)((s.pos + t - back) % g.width) * g.channels + c]);
            v = fmaf(g.weight[(size_t)k * g.channels + c], u, v);
        }
        static_cast<T *>(g.out)[(size_t)row * g.ldo + c] = from_f32<T>(g.silu ? silu(v) : v);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void k_conv_ring_simple(mdf_conv_args g)
{
    const Seq s = seq_of(g.rows, blockIdx.x, true);
    T *ring = static_cast<T *>(g.state) + (size_t)s.slot * g.width * g.channels;
    for (int t = max(0, s.count - g.width); t < s.count; ++t)
        for (int c = threadIdx.x; c < g.channels; c += 256)
            ring[(size_t)((s.pos + t) % g.width) * g.channels + c] = static_cast<const T *>(g.x)[(size_t)(s.row + t) * g.ldx + c];
}

// ---- the selective scan: simple form, one workgroup per sequence, head and 64 channels, the state in LDS ---------------------------------
template <typename T>
__global__ __launch_bounds__(64) void k_scan_simple(mdf_scan_args g)
{
    __shared__ float H[64][129];
    __shared__ float B[128], C[128];
    const int h = blockIdx.y, p = blockIdx.z * 64 + threadIdx.x, grp = h / (g.heads / g.groups), N = g.state_dim;
    const Seq s = seq_of(g.rows, blockIdx.x, g.state != nullptr);
    if (s.count < 0) return;
    const bool on = p < g.head_dim;
    float *st = g.state ? g.state + (((size_t)s.slot * g.heads + h) * g.head_dim + p) * N : nullptr;
    for (int n = 0; n < N; ++n) H[threadIdx.x][n] = on && st && s.pos > 0 ? st[n] : 0.0f;
    for (int t = 0; t < s.count; ++t) {
        const size_t row = (size_t)(s.row + t);
        __syncthreads();
        for (int n = threadIdx.x; n < N; n += 64) {
            B[n] = to_f32(static_cast<const T *>(g.b)[row * g.ldb + grp * N + n]);
            C[n] = to_f32(static_cast<const T *>(g.c)[row * g.ldc + grp * N + n]);
        }
        __syncthreads();
        if (!on) continue;
        const float delta = softplus(load_any(g.dt, row * g.lddt + h, g.dt_dtype) + (g.dt_bias ? g.dt_bias[h] : 0.0f));
        const float decay = expf(delta * g.a[h]), x = to_f32(static_cast<const T *>(g.x)[row * g.ldx + (size_t)h * g.head_dim + p]), u = delta * x;
        float y = 0.0f;
        for (int n = 0; n < N; ++n) {
            const float v = fmaf(decay, H[threadIdx.x][n], u * B[n]);
            H[threadIdx.x][n] = v;
            y = fmaf(v, C[n], y);
        }
        if (g.d) y = fmaf(g.d[h], x, y);
        static_cast<T *>(g.y)[row * g.ldy + (size_t)h * g.head_dim + p] = from_f32<T>(y);
    }
    if (on && st && s.count > 0)
        for (int n = 0; n < N; ++n) st[n] = H[threadIdx.x][n];
}

// ---- one token: simple form, one workgroup per sequence and head ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_step_simple(mdf_step_args g)
{
    __shared__ float u[256 + 2 * 128];   // the head's x, B, C after the convolution
    const int b = blockIdx.x, h = blockIdx.y, r = g.heads / g.groups, grp = h / r, P = g.head_dim, N = g.state_dim, W = g.width;
    const int slot = g.slots ? g.slots[b] : b;
    if (slot < 0 || slot >= g.n_slots) return;
    const int64_t pos = g.positions ? max(g.positions[b], 0) : 0;
    const int channels = g.heads * P + 2 * g.groups * N;
    T *ring = static_cast<T *>(g.conv_state) + (size_t)slot * W * channels;
    for (int i = threadIdx.x; i < P + 2 * N; i += 256) {
        const int c = i < P ? h * P + i : i < P + N ? g.heads * P + grp * N + i - P : g.heads * P + (g.groups + grp) * N + i - P - N;
        const T now = static_cast<const T *>(g.xbc)[(size_t)b * g.ldx + c];
        float v = g.conv_bias ? g.conv_bias[c] : 0.0f;
        for (int back = W - 1; back > 0; --back)
            if (pos >= back) v = fmaf(g.conv_weight[(size_t)(W - 1 - back) * channels + c], to_f32(ring[(size_t)((pos - back) % W) * channels + c]), v);
        v = fmaf(g.conv_weight[(size_t)(W - 1) * channels + c], to_f32(now), v);
        u[i] = silu(v);
        if (i < P || h % r == 0) ring[(size_t)(pos % W) * channels + c] = now;   // an entry that no workgroup of this launch reads
    }
    __syncthreads();
    const float delta = softplus(load_any(g.dt, (size_t)b * g.lddt + h, g.dt_dtype) + (g.dt_bias ? g.dt_bias[h] : 0.0f)), decay = expf(delta * g.a[h]);
    for (int p = threadIdx.x; p < P; p += 256) {
        float *st = g.state + (((size_t)slot * g.heads + h) * P + p) * N;
        float y = g.d ? g.d[h] * u[p] : 0.0f;
        for (int n = 0; n < N; ++n) {
            const float v = fmaf(decay, pos > 0 ? st[n] : 0.0f, delta * u[p] * u[P + n]);
            st[n] = v;
            y = fmaf(v, u[P + N + n], y);
        }
        static_cast<T *>(g.y)[(size_t)b * g.ldy + (size_t)h * P + p] = from_f32<T>(y);
    }
}

// ---- block norms: simple form, one workgroup per row and group, three walks over the row ------------------------------------------------------
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
__global__ __launch_bounds__(256) void k_block_norm_simple(mdf_block_norm_args g)
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
    float m1 = 0.0f, q1 = 1.0f, m2 = 0.0f, q2 = 1.0f, sum = 0.0f;
    if (g.post_weight) {
        if (g.center) {
            for (int c = c0 + threadIdx.x; c < c1; c += 256) sum += first(c);
            m1 = block_sum(sum) / width;
        }
        sum = 0.0f;
        for (int c = c0 + threadIdx.x; c < c1; c += 256) sum += (first(c) - m1) * (first(c) - m1);
        q1 = 1.0f / sqrtf(block_sum(sum) / width + g.eps);
    }
    auto after = [&](int c) {
        float v = first(c);
        if (g.post_weight) v = (v - m1) * q1 * g.post_weight[c] + (g.post_bias ? g.post_bias[c] : 0.0f);
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
        q2 = 1.0f / sqrtf(block_sum(sum) / width + g.eps);
    }
    for (int c = c0 + threadIdx.x; c < c1; c += 256) {
        const float v = after(c);
        if (res) static_cast<R *>(g.residual_out)[row * g.ldro + c] = from_f32<R>(v);
        if (g.pre_weight) static_cast<T *>(g.out)[row * g.ldo + c] = from_f32<T>((v - m2) * q2 * g.pre_weight[c] + (g.pre_bias ? g.pre_bias[c] : 0.0f));
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
    if (int rc = require_device()) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    MDF_BY_TYPE(a->dtype, T, {
        hipLaunchKernelGGL(k_conv_simple<T>, dim3((unsigned)a->rows.R), dim3(256), 0, st, *a);
        if (a->state) hipLaunchKernelGGL(k_conv_ring_simple<T>, dim3((unsigned)a->rows.B), dim3(256), 0, st, *a);
    });
    MDF_HIP(hipGetLastError());
    return MDF_OK;
}

size_t mdf_scan_workspace_bytes(const mdf_scan_args *) { return 0; }

int mdf_selective_scan_dev(const mdf_scan_args *a, void *, size_t, void *stream)
{
    MDF_REQUIRE(a, "selective_scan_dev: NULL argument");
    if (int rc = check_rows(a->rows, "selective_scan_dev", a->state != nullptr)) return rc;
    MDF_REQUIRE(dt_size(a->dtype) && dt_size(a->dt_dtype), "selective_scan_dev: dtype %d / %d is not f32, bf16 or f16", a->dtype, a->dt_dtype);
    MDF_REQUIRE(a->heads > 0 && a->heads <= 65535 && a->groups > 0 && a->heads % a->groups == 0, "selective_scan_dev: %d heads in %d groups", a->heads, a->groups);
    MDF_REQUIRE(a->head_dim >= 1 && a->head_dim <= 256 && a->state_dim >= 1 && a->state_dim <= 128, "selective_scan_dev: head_dim=%d (1..256), state_dim=%d (1..128)",
                a->head_dim, a->state_dim);
    if (a->rows.B == 0 || (a->rows.R == 0 && !a->state)) return MDF_OK;
    MDF_REQUIRE((a->x && a->b && a->c && a->dt && a->y) || a->rows.R == 0, "selective_scan_dev: NULL argument");
    MDF_REQUIRE(a->a, "selective_scan_dev: a is NULL");
    const int64_t R = a->rows.R, hp = (int64_t)a->heads * a->head_dim, gn = (int64_t)a->groups * a->state_dim;
    MDF_REQUIRE(a->ldx >= 0 && a->ldb >= 0 && a->ldc >= 0 && a->lddt >= 0 && (a->ldy >= hp || R <= 1), "selective_scan_dev: a row stride is negative or y's is below %lld", (long long)hp);
    const size_t e = dt_size(a->dtype);
    MDF_REQUIRE(!overlap(a->x, a->ldx, hp, e, a->y, a->ldy, hp, e, R) && !overlap(a->b, a->ldb, gn, e, a->y, a->ldy, hp, e, R) &&
                    !overlap(a->c, a->ldc, gn, e, a->y, a->ldy, hp, e, R) && !overlap(a->dt, a->lddt, a->heads, dt_size(a->dt_dtype), a->y, a->ldy, hp, e, R),
                "selective_scan_dev: y overlaps an input");
    if (int rc = require_device()) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    MDF_BY_TYPE(a->dtype, T, hipLaunchKernelGGL(k_scan_simple<T>, dim3((unsigned)a->rows.B, a->heads, (a->head_dim + 63) / 64), dim3(64), 0, st, *a));
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
    MDF_BY_TYPE(a->dtype, T, hipLaunchKernelGGL(k_step_simple<T>, dim3(a->B, a->heads), dim3(256), 0, st, *a));
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
    MDF_BY_TYPE(a->dtype, T, {
        if (a->residual && a->residual_dtype == MDF_DT_F32) hipLaunchKernelGGL((k_block_norm_simple<T, float>), dim3((unsigned)a->rows, a->groups), dim3(256), 0, st, *a);
        else hipLaunchKernelGGL((k_block_norm_simple<T, T>), dim3((unsigned)a->rows, a->groups), dim3(256), 0, st, *a);
    });
    MDF_HIP(hipGetLastError());
    return MDF_OK;
}

}  // extern "C"
