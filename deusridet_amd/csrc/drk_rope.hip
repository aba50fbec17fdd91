// drk_rope.hip -- rotary positions for long contexts: frequencies stretched per pair, either
// pair layout, part of a head, strided rows, both directions.
//
// For a pair (a, b) of a head at position p, with f its turns per position and m the magnitude:
//   a' = m (a cos w - b sin w),  b' = m (b cos w + a sin w),  w = 2 pi p f
// (inverse: sin w with the other sign -- the transpose, which is the gradient).  p f is formed in
// 64 bits and only its fraction of a turn goes on in 32 bits: in 32 bits the angle of position
// 10^6 would carry an error of 0.06 rad.  The hardware's sine and cosine take turns, so no range
// reduction follows; their error, about 2^-20, is far below the 16-bit result's rounding.
//
// Bound by HBM: 4 bytes an element.  8192 tokens x 40 heads x 128 (168 MB): 32 us, 5.2 TB/s read and written, where
// torch's copy of as many bytes takes 36; every row is touched once, hence non-temporal loads and stores.  A decode
// step (64 tokens x 28 heads x 256) is a launch and one round trip to memory: 3.8 us.
#include "drk_common.hpp"
#include "drk_codec.hpp"

#include <math.h>

namespace drk {

constexpr int kRThreads = 256;
// Threads from which one takes four head rows: above, the sines are formed once for four (8192 tokens 33.3 us, one row each
// 35.4); below, more threads hide the round trip better (64 tokens 6.9 us through the entry point, four rows each 7.4).
constexpr size_t kRopeShare = 1 << 18;

// f'_i, see drk_rope in drk_kv.h
__device__ __forceinline__ double rope_turns(const drk_rope &r, int i)
{
    const double f = pow((double)r.theta, -2.0 * i / r.rotary_dim) * 0.15915494309189533577;   // 1 / (2 pi)
    if (r.factor == 1.0f) return f;
    double g = (f * r.original_positions - r.low_turns) / ((double)r.high_turns - r.low_turns);
    g = g < 0.0 ? 0.0 : (g > 1.0 ? 1.0 : g);
    return f * (g + (1.0 - g) / r.factor);
}

// cos and sin of p f turns
__device__ __forceinline__ void rope_cos_sin(double p, double f, float &c, float &s)
{
    const double w = p * f;
    const float x = (float)(w - floor(w));
#if defined(__HIP_DEVICE_COMPILE__)
    c = __builtin_amdgcn_cosf(x);
    s = __builtin_amdgcn_sinf(x);
#else
    c = x;
    s = x;
#endif
}

__global__ __launch_bounds__(kRThreads) void rope_freqs_kernel(drk_rope r, double *__restrict__ freqs)
{
    const int i = blockIdx.x * kRThreads + threadIdx.x;
    if (i < r.rotary_dim / 2) freqs[i] = rope_turns(r, i);
}

__global__ __launch_bounds__(kRThreads) void rope_table_scaled_kernel(drk_rope r, float *__restrict__ table, int n_pos)
{
    const int np = r.rotary_dim / 2;
    const size_t i = (size_t)blockIdx.x * kRThreads + threadIdx.x;
    if (i >= (size_t)n_pos * np) return;
    const int pos = (int)(i / np), pair = (int)(i - (size_t)pos * np);
    const double w = pos * rope_turns(r, pair);
    const double x = (w - floor(w)) * 6.28318530717958647693;
    *(float2 *)(table + i * 2) = make_float2((float)(cos(x) * r.magnitude), (float)(sin(x) * r.magnitude));
}

struct RopeArgs {
    drk_rope_rows tensors[DRK_ROPE_MAX_TENSORS];
    const double *freqs;
    const int32_t *d_pos;
    int first_head[DRK_ROPE_MAX_TENSORS];   // head rows before tensor i in a token's list of them
    int n_tensors, pos_start, T, rows, row_groups, units, hp, interleaved;
    float cm, sm;                           // factors of cos and sin: the magnitude, and its sign turned for the inverse
};

__device__ __forceinline__ uint4 rope_pack8(const float *y, int dtype)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (dtype == DRK_BF16)
            w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)y[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)y[2 * i + 1]) << 16);
        else
            w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y[2 * i + 1]) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// One thread: 8 pairs (or 16 elements that pass unchanged) of HPT head rows of one token, whose angles are the
// same: the sines, about half of the arithmetic of a row by itself, are formed once.  The heads of a token are
// taken HPT-strided groups apart, so that neighbouring lanes stay on neighbouring bytes.
template <int HPT, int DTYPE>
__global__ __launch_bounds__(kRThreads) void rope_apply_kernel(RopeArgs A)
{
    const size_t it = (size_t)blockIdx.x * kRThreads + threadIdx.x;
    if (it >= (size_t)A.T * A.row_groups * A.units) return;
    const size_t row = it / A.units;
    const int u = (int)(it - row * A.units);
    const int t = (int)(row / A.row_groups), h0 = (int)(row - (size_t)t * A.row_groups);
    const bool rotated = u < A.hp;
    // chunks u and u + hp of 8 elements: half-half, pair (i, i + r/2), they are 8 pairs; interleaved 4 pairs each.  Behind the
    // rotary part likewise.  Neighbouring lanes are on neighbouring chunks in both accesses.
    const int e0 = rotated ? u * 8 : A.hp * 16 + (u - A.hp) * 8, e1 = e0 + (rotated ? A.hp : A.units - A.hp) * 8;
    uint4 va[HPT], vb[HPT];
    uint16_t *o[HPT];
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        int h = h0 + i * A.row_groups, n = 0;
        if (h >= A.rows) { o[i] = nullptr; continue; }
        while (n + 1 < A.n_tensors && h >= A.first_head[n + 1]) n++;
        h -= A.first_head[n];
        const drk_rope_rows &R = A.tensors[n];
        const uint16_t *x = (const uint16_t *)R.x + (size_t)t * R.x_token_stride + (size_t)h * R.x_head_stride;
        o[i] = (uint16_t *)R.out + (size_t)t * R.out_token_stride + (size_t)h * R.out_head_stride;
        va[i] = ld_stream128(x + e0);
        vb[i] = ld_stream128(x + e1);
    }
    float c[8], s[8];
    if (rotated) {
        const double p = A.d_pos ? A.d_pos[t] : (double)A.pos_start + t;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            rope_cos_sin(p, A.freqs[A.interleaved ? (i < 4 ? u : u + A.hp - 1) * 4 + i : u * 8 + i], c[i], s[i]);
            c[i] *= A.cm;
            s[i] *= A.sm;
        }
    }
#pragma unroll
    for (int k = 0; k < HPT; k++) {
        if (!o[k]) continue;
        if (rotated) {
            float a[8], b[8], y0[8], y1[8];
            unpack8(va[k], DTYPE, a);
            unpack8(vb[k], DTYPE, b);
            if (A.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    y0[2 * i] = a[2 * i] * c[i] - a[2 * i + 1] * s[i];
                    y0[2 * i + 1] = a[2 * i + 1] * c[i] + a[2 * i] * s[i];
                    y1[2 * i] = b[2 * i] * c[i + 4] - b[2 * i + 1] * s[i + 4];
                    y1[2 * i + 1] = b[2 * i + 1] * c[i + 4] + b[2 * i] * s[i + 4];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    y0[i] = a[i] * c[i] - b[i] * s[i];
                    y1[i] = b[i] * c[i] + a[i] * s[i];
                }
            }
            va[k] = rope_pack8(y0, DTYPE);
            vb[k] = rope_pack8(y1, DTYPE);
        }
        st_stream128(o[k] + e0, va[k]);
        st_stream128(o[k] + e1, vb[k]);
    }
}

static int check_rope(const drk_rope *r, const char *who)
{
    if (!r) return fail(DRK_ERR_INVALID, "%s: NULL description", who);
    if (r->rotary_dim < 16 || (r->rotary_dim % 16))
        return fail(DRK_ERR_UNSUPPORTED, "%s: rotary_dim %d must be a multiple of 16", who, r->rotary_dim);
    if (r->interleaved != 0 && r->interleaved != 1) return fail(DRK_ERR_INVALID, "%s: interleaved must be 0 or 1", who);
    if (!(r->theta > 0.0f) || !isfinite(r->theta) || !(r->factor > 0.0f) || !isfinite(r->factor) || !isfinite(r->magnitude))
        return fail(DRK_ERR_INVALID, "%s: theta and factor must be positive, magnitude finite", who);
    if (r->factor != 1.0f && !(r->original_positions >= 0.0f && r->low_turns >= 0.0f && r->high_turns > r->low_turns &&
                               isfinite(r->original_positions) && isfinite(r->high_turns)))
        return fail(DRK_ERR_INVALID, "%s: original_positions >= 0 and 0 <= low_turns < high_turns are wanted", who);
    return DRK_OK;
}

} // namespace drk

using namespace drk;

extern "C" {

int drk_rope_freqs_fill(const drk_rope *r, double *d_freqs, void *stream)
{
    int rc = check_rope(r, "rope_freqs_fill");
    if (rc) return rc;
    if (!d_freqs) return fail(DRK_ERR_INVALID, "rope_freqs_fill: NULL pointer");
    hipLaunchKernelGGL(rope_freqs_kernel, dim3((r->rotary_dim / 2 + kRThreads - 1) / kRThreads), dim3(kRThreads), 0,
                       (hipStream_t)stream, *r, d_freqs);
    DRK_LAUNCH_CHECK("rope_freqs_kernel");
    return DRK_OK;
}

int drk_rope_table_fill_scaled(const drk_rope *r, float *d_table, int n_pos, void *stream)
{
    int rc = check_rope(r, "rope_table_fill_scaled");
    if (rc) return rc;
    if (!d_table || n_pos < 1) return fail(DRK_ERR_INVALID, "rope_table_fill_scaled: bad argument");
    if (r->interleaved) return fail(DRK_ERR_UNSUPPORTED, "rope_table_fill_scaled: the entry points that read a table rotate half-half pairs");
    const size_t blocks = ((size_t)n_pos * (r->rotary_dim / 2) + kRThreads - 1) / kRThreads;
    if (blocks > 0x7fffffffu) return fail(DRK_ERR_INVALID, "rope_table_fill_scaled: table too large");
    hipLaunchKernelGGL(rope_table_scaled_kernel, dim3((unsigned)blocks), dim3(kRThreads), 0, (hipStream_t)stream, *r, d_table, n_pos);
    DRK_LAUNCH_CHECK("rope_table_scaled_kernel");
    return DRK_OK;
}

int drk_rope_apply(const drk_rope *r, const double *d_freqs, const drk_rope_rows *tensors, int n_tensors, int T, int head_dim,
                   const int32_t *d_pos, int pos_start, int inverse, int dtype, void *stream)
{
    int rc = check_rope(r, "rope_apply");
    if (rc) return rc;
    if (dtype != DRK_F16 && dtype != DRK_BF16) return fail(DRK_ERR_INVALID, "rope_apply: dtype must be F16 or BF16");
    if (head_dim < 16 || head_dim > 1024 || (head_dim % 16) || r->rotary_dim > head_dim)
        return fail(DRK_ERR_UNSUPPORTED, "rope_apply: head_dim %d must be a multiple of 16 up to 1024, rotary_dim %d at most that",
                    head_dim, r->rotary_dim);
    if (!d_freqs || !tensors || n_tensors < 1 || n_tensors > DRK_ROPE_MAX_TENSORS || T < 0 || pos_start < 0)
        return fail(DRK_ERR_INVALID, "rope_apply: bad argument");
    RopeArgs A;
    A.rows = 0;
    bool in_place = true;
    for (int i = 0; i < n_tensors; i++) {
        const drk_rope_rows &x = tensors[i];
        if (x.heads < 0 || x.reserved != 0 || (x.heads > 0 && T > 0 && (!x.x || !x.out)))
            return fail(DRK_ERR_INVALID, "rope_apply: tensor %d: bad argument", i);
        if (((uintptr_t)x.x | (uintptr_t)x.out) & 15u || (x.x_token_stride | x.x_head_stride | x.out_token_stride | x.out_head_stride) & 7u)
            return fail(DRK_ERR_INVALID, "rope_apply: tensor %d: pointers must be 16-byte aligned, strides multiples of 8", i);
        if (x.heads > 1 && x.out_head_stride < (size_t)head_dim)
            return fail(DRK_ERR_INVALID, "rope_apply: tensor %d: heads of out overlap", i);
        // rows of out are written by different threads: tokens behind one another's heads, or heads behind one another's tokens
        if (x.heads > 0 && T > 1 && x.out_token_stride < (size_t)(x.heads - 1) * x.out_head_stride + head_dim &&
            (x.out_token_stride < (size_t)head_dim || x.heads == 1 || x.out_head_stride < (size_t)(T - 1) * x.out_token_stride + head_dim))
            return fail(DRK_ERR_INVALID, "rope_apply: tensor %d: rows of out overlap", i);
        for (int j = 0; j < i; j++) {
            if (x.heads <= 0 || tensors[j].heads <= 0) continue;
            if (x.out == tensors[j].out) return fail(DRK_ERR_INVALID, "rope_apply: tensors %d and %d have one output", j, i);
            // the tensors are rotated side by side: what one writes another must not read
            if (x.out == tensors[j].x || x.x == tensors[j].out)
                return fail(DRK_ERR_INVALID, "rope_apply: of tensors %d and %d one reads what the other writes", j, i);
        }
        if (x.x == x.out && (x.x_token_stride != x.out_token_stride || x.x_head_stride != x.out_head_stride))
            return fail(DRK_ERR_INVALID, "rope_apply: tensor %d: in place needs equal strides", i);
        if (x.heads > (1 << 20)) return fail(DRK_ERR_INVALID, "rope_apply: tensor %d: %d heads", i, x.heads);
        in_place = in_place && x.x == x.out;
        A.tensors[i] = x;
        A.first_head[i] = A.rows;
        A.rows += x.heads;
    }
    A.freqs = d_freqs; A.d_pos = d_pos; A.n_tensors = n_tensors; A.pos_start = pos_start; A.T = T;
    A.hp = r->rotary_dim / 16;
    A.units = in_place ? A.hp : head_dim / 16;              // in place, what passes unchanged is there already
    A.interleaved = r->interleaved;
    A.cm = r->magnitude; A.sm = inverse ? -r->magnitude : r->magnitude;
    const size_t all = (size_t)T * A.rows * A.units;
    if (all == 0) return DRK_OK;
    const int hpt = all >= kRopeShare ? 4 : 1;
    A.row_groups = (A.rows + hpt - 1) / hpt;
    const size_t blocks = ((size_t)T * A.row_groups * A.units + kRThreads - 1) / kRThreads;
    if (blocks > 0x7fffffffu) return fail(DRK_ERR_INVALID, "rope_apply: too many rows");
    const dim3 grid((unsigned)blocks);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DRK_BF16) {
        if (hpt == 4) hipLaunchKernelGGL((rope_apply_kernel<4, DRK_BF16>), grid, dim3(kRThreads), 0, st, A);
        else hipLaunchKernelGGL((rope_apply_kernel<1, DRK_BF16>), grid, dim3(kRThreads), 0, st, A);
    } else {
        if (hpt == 4) hipLaunchKernelGGL((rope_apply_kernel<4, DRK_F16>), grid, dim3(kRThreads), 0, st, A);
        else hipLaunchKernelGGL((rope_apply_kernel<1, DRK_F16>), grid, dim3(kRThreads), 0, st, A);
    }
    DRK_LAUNCH_CHECK("rope_apply_kernel");
    return DRK_OK;
}

} // extern "C"
