// drk_bounds.hip -- bounds of every block's keys: for each (layer, physical block, kv head) the
// lowest and highest key per dimension, as int8 codes of one power of two.
//
// The code of a bound is floor(low / 2^e) or ceil(high / 2^e) with e from the block's largest
// magnitude: scaling by a power of two is exact, so the codes follow from the keys alone, without
// a rounding that could depend on an order.  All of it is HBM-bound: a key row is read once, 2 D + 1
// bytes come back per block and head.  16 layers x 9 blocks of 256 tokens x 4 heads x 256 in f16 (75 MB): 16 us, 4.7 TB/s,
// of which 4 are the launch and the first round trip; 131 072 int8 tokens x 8 heads x 128 in blocks of 16 (153 MB): 31 us,
// 4.9 TB/s -- about 1450 vector instructions a thread, 20 us of a SIMD's time, run in the shadow of the loads only in part
// (a sixth of them taken out changed nothing).  One decode step of 8 branches: 3.5 us, the launch and three dependent loads.
#include "drk_common.hpp"
#include "drk_codec.hpp"
#include "drk_bounds.hpp"

namespace drk {

constexpr int kBThreads = 256;
// Which kernel: a thread takes 16 bytes of every row of its (layer, block, kv head), one row after the other (short), or a
// workgroup takes the rows 16 per thread at once and folds in LDS (long).  The first takes as long as a block has rows, the
// second as long as there are units, for 64 KiB of loads each, those beyond the unit's last row repeated.  Us, short / long:
//   few units, 8 branches x 8 heads:  bf16 x 128, blocks of 32 4.3 / 4.3, 64 6.0 / 4.2, 256 16.7 / 4.2; int8 32 7.4 / 7.1, 64 11.9 / 7.1
//   131 072 tokens x 8 heads, int8 x 128:  blocks of 32 26 / 398, 64 24 / 205, 128 30 / 105, 256 52 / 61
//   65 536 tokens x 8 heads, bf16 x 128:   blocks of 32 22 / 64, 64 21 / 32, 128 22 / 22, 256 31 / 21
// So: the long one for blocks above 32 tokens where the units are fewer than a unit's 16-byte chunks, or a unit fills the loads.
constexpr int kBLongBlock = 32;
constexpr size_t kBLongBytes = 64 << 10;

struct BoundsArgs {
    const uint8_t *pool;
    uint8_t *bounds;
    const int32_t *tables, *d_pos;
    size_t exps;                   // offset of the exponents in the buffer
    int table_stride, pos_start, n, first_block, n_blocks, layer0;
    unsigned units;                // (layer, block, kv head) triples
    Div bs_div;
};

// 16 bytes of a key row as floats
template <int DT> struct BoundsElems { static constexpr int V = 8; };
template <> struct BoundsElems<DRK_INT8> { static constexpr int V = 16; };
template <> struct BoundsElems<DRK_FP8_E4M3> { static constexpr int V = 16; };
template <int DT>
__device__ __forceinline__ void bounds_unpack(const uint4 &v, float scale, float *x)
{
    if constexpr (DT == DRK_F16 || DT == DRK_BF16) {
        unpack8(v, DT, x);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == DRK_INT8) {
                // (code + 128) scale - 128 scale, rounded once: code * scale, exactly (a byte becomes a float in one
                // instruction only if it is unsigned); a scale that is not finite gives NaN, which is passed over
                const uint32_t u = w[i] ^ 0x80808080u;
#pragma unroll
                for (int j = 0; j < 4; j++) x[4 * i + j] = __fmaf_rn((float)(u >> (8 * j) & 0xffu), scale, -128.0f * scale);
            } else {
                uint32_t lo, hi;
                fp8x4_to_f16x4(w[i], lo, hi);
                x[4 * i] = f16_bits_to_f((uint16_t)(lo & 0xffffu));
                x[4 * i + 1] = f16_bits_to_f((uint16_t)(lo >> 16));
                x[4 * i + 2] = f16_bits_to_f((uint16_t)(hi & 0xffffu));
                x[4 * i + 3] = f16_bits_to_f((uint16_t)(hi >> 16));
            }
        }
    }
}

// a (layer, block, kv head): where its keys are and how many of them count
struct BoundsUnit { int layer, blk, cnt; unsigned h; };
__device__ __forceinline__ BoundsUnit bounds_unit(const Lay &a, const BoundsArgs &A, unsigned unit)
{
    BoundsUnit U;
    const unsigned rest = unit / (unsigned)a.KVH, bi = rest % (unsigned)A.n_blocks;
    U.h = unit - rest * (unsigned)a.KVH;
    U.layer = A.layer0 + (int)(rest / (unsigned)A.n_blocks);
    U.blk = -1;
    U.cnt = 0;
    const int32_t *tab = A.tables;
    int pos, lb;
    if (A.d_pos) {
        pos = A.d_pos[bi];
        lb = pos < 0 ? -1 : (int)dv((unsigned)pos, A.bs_div);
        tab += (size_t)bi * A.table_stride;
        if (A.table_stride > 0 && lb >= A.table_stride) lb = -1;       // stride 0: one table for all, as long as its positions need
    } else {
        lb = A.first_block + (int)bi;
        pos = A.pos_start + A.n - 1;
    }
    if (lb < 0) return U;
    U.blk = tab[lb];
    if (U.blk >= 0 && U.blk < a.NB) U.cnt = min(a.bs, pos - lb * a.bs + 1);
    return U;
}

// everything above is issued before anything below: the compiler would trade loads in flight for registers
__device__ __forceinline__ void bounds_issue_barrier()
{
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_barrier(0);
#endif
}

// lowest and highest of 16 bytes of each of the rows r0, r0 + step, .. of a unit; B rows in flight
template <int DT, int B>
__device__ __forceinline__ void bounds_rows(const Lay &a, const BoundsArgs &A, const BoundsUnit &U, unsigned sub, int r0, int step,
                                            float *lo, float *hi)
{
    constexpr int V = BoundsElems<DT>::V;
#pragma unroll
    for (int i = 0; i < V; i++) { lo[i] = INFINITY; hi[i] = -INFINITY; }
    if (r0 >= U.cnt) return;
    const uint8_t *base = A.pool + row_off(a, U.layer, U.blk, 0, (int)U.h, 0) + sub * 16;
    const uint8_t *sc = A.pool + (DT == DRK_INT8 ? scale_off(a, U.layer, U.blk, 0, (int)U.h, 0) : 0);
    for (int r = r0; r < U.cnt; r += B * step) {
        uint4 v[B];
        float s[B];
#pragma unroll
        for (int u = 0; u < B; u++) {
            const int rr = min(r + u * step, U.cnt - 1);               // a row read twice changes no bound
            v[u] = ld_stream128(base + (size_t)rr * a.row_bytes);
            s[u] = DT == DRK_INT8 ? f16_bits_to_f(*(const uint16_t *)(sc + (size_t)rr * 2)) : 1.0f;
        }
        bounds_issue_barrier();
#pragma unroll
        for (int u = 0; u < B; u += 2) {                               // two rows at a time: three-way minimum and maximum
            float x[V], y[V];
            bounds_unpack<DT>(v[u], s[u], x);
            bounds_unpack<DT>(v[u + 1], s[u + 1], y);
#pragma unroll
            for (int i = 0; i < V; i++) { lo[i] = fminf(fminf(lo[i], x[i]), y[i]); hi[i] = fmaxf(fmaxf(hi[i], x[i]), y[i]); }
        }
    }
}

__device__ __forceinline__ uint32_t bounds_code(float x, int e, bool high)
{
    const float y = fminf(fmaxf(ldexpf(x, -e), -127.0f), 127.0f);
    return (uint32_t)(int)(high ? ceilf(y) : floorf(y)) & 0xffu;
}

// Many or short units: a thread owns 16 bytes of every row of its unit, so nothing is exchanged but the largest magnitude;
// row_bytes / 16 neighbouring lanes hold a unit.
template <int DT>
__global__ __launch_bounds__(kBThreads) void bounds_update_kernel(Lay a, BoundsArgs A, unsigned lpr, int lpr_shift)
{
    constexpr int V = BoundsElems<DT>::V;
    const size_t i0 = (size_t)blockIdx.x * kBThreads + threadIdx.x;
    const size_t unit = i0 >> lpr_shift;
    const unsigned sub = (unsigned)i0 & (lpr - 1);
    BoundsUnit U = {0, -1, 0, 0};
    if (unit < A.units) U = bounds_unit(a, A, (unsigned)unit);
    float lo[V], hi[V];
    bounds_rows<DT, 8>(a, A, U, sub, 0, 1, lo, hi);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (lo[i] > hi[i]) lo[i] = hi[i] = 0.0f;                       // nothing but NaN
        amax = fmaxf(amax, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
    }
    for (unsigned off = lpr >> 1; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, (int)off));
    if (U.cnt <= 0) return;
    const int e = bounds_exponent(amax);
    uint32_t cl[V / 4], ch[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        cl[i] = ch[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            cl[i] |= bounds_code(lo[4 * i + j], e, false) << (8 * j);
            ch[i] |= bounds_code(hi[4 * i + j], e, true) << (8 * j);
        }
    }
    const size_t entry = ((size_t)U.layer * a.NB + U.blk) * a.KVH + U.h;
    uint8_t *dst = A.bounds + entry * 2 * a.D + sub * V;
    if constexpr (V == 8) {
        *(uint2 *)dst = make_uint2(cl[0], cl[1]);
        *(uint2 *)(dst + a.D) = make_uint2(ch[0], ch[1]);
    } else {
        *(uint4 *)dst = make_uint4(cl[0], cl[1], cl[2], cl[3]);
        *(uint4 *)(dst + a.D) = make_uint4(ch[0], ch[1], ch[2], ch[3]);
    }
    if (sub == 0) A.bounds[A.exps + entry] = (uint8_t)(int8_t)e;
}

// Few or long units: a workgroup per unit, its rows dealt out to 256 / lpr threads per 16-byte column; the partial bounds meet
// in LDS, where thread d then owns dimension d.
template <int DT>
__global__ __launch_bounds__(kBThreads) void bounds_update_long_kernel(Lay a, BoundsArgs A, unsigned lpr, int lpr_shift)
{
    constexpr int V = BoundsElems<DT>::V;
    __shared__ __align__(16) float red[2][kBThreads * V];              // [low, high][row group][dimension]
    __shared__ float wmax[4];
    const BoundsUnit U = bounds_unit(a, A, blockIdx.x);
    if (U.cnt <= 0) return;                                            // the same for the whole workgroup
    const unsigned sub = threadIdx.x & (lpr - 1), rg = threadIdx.x >> lpr_shift;
    const int groups = (int)(kBThreads >> lpr_shift);
    float lo[V], hi[V];
    bounds_rows<DT, 16>(a, A, U, sub, (int)rg, groups, lo, hi);
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        *(float4 *)&red[0][rg * a.D + sub * V + i] = make_float4(lo[i], lo[i + 1], lo[i + 2], lo[i + 3]);
        *(float4 *)&red[1][rg * a.D + sub * V + i] = make_float4(hi[i], hi[i + 1], hi[i + 2], hi[i + 3]);
    }
    __syncthreads();
    float l[2], g[2], amax = 0.0f;                                     // head_dim is at most 512
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int d = (int)threadIdx.x + k * kBThreads;
        l[k] = INFINITY;
        g[k] = -INFINITY;
        if (d >= a.D) continue;
        for (int r = 0; r < groups; r++) { l[k] = fminf(l[k], red[0][r * a.D + d]); g[k] = fmaxf(g[k], red[1][r * a.D + d]); }
        if (l[k] > g[k]) l[k] = g[k] = 0.0f;
        amax = fmaxf(amax, fmaxf(fabsf(l[k]), fabsf(g[k])));
    }
    for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
    if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = amax;
    __syncthreads();
    const int e = bounds_exponent(fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3])));
    const size_t entry = ((size_t)U.layer * a.NB + U.blk) * a.KVH + U.h;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int d = (int)threadIdx.x + k * kBThreads;
        if (d >= a.D) continue;
        A.bounds[entry * 2 * a.D + d] = (uint8_t)bounds_code(l[k], e, false);
        A.bounds[entry * 2 * a.D + a.D + d] = (uint8_t)bounds_code(g[k], e, true);
    }
    if (threadIdx.x == 0) A.bounds[A.exps + entry] = (uint8_t)(int8_t)e;
}

// 16 codes per thread -> 16 bf16 values (7 bits and a power of two: exact)
__global__ __launch_bounds__(kBThreads) void bounds_extract_kernel(Lay a, uint8_t *__restrict__ dst, const uint8_t *__restrict__ bounds,
                                                                  size_t exps, const int32_t *__restrict__ blocks, int n_blocks,
                                                                  int layer0, size_t chunks, int cps)
{
    const size_t i = (size_t)blockIdx.x * kBThreads + threadIdx.x;
    if (i >= chunks) return;
    const size_t row = i >> cps;                                     // (layer, block, head)
    const unsigned c = (unsigned)(i & ((1u << cps) - 1));
    const unsigned h = (unsigned)(row % a.KVH);
    const size_t lb = row / a.KVH;
    const int layer = layer0 + (int)(lb / n_blocks), blk = blocks[lb % n_blocks];
    uint4 o[2] = {};
    if (blk >= 0 && blk < a.NB) {
        const size_t entry = ((size_t)layer * a.NB + blk) * a.KVH + h;
        const uint4 v = *(const uint4 *)(bounds + entry * 2 * a.D + c * 16);
        const float s = ldexpf(1.0f, (int)(int8_t)bounds[exps + entry]);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t y[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float x0 = (float)(int8_t)(w[k / 2] >> (16 * (k & 1))) * s, x1 = (float)(int8_t)(w[k / 2] >> (16 * (k & 1) + 8)) * s;
            y[k] = (__float_as_uint(x0) >> 16) | (__float_as_uint(x1) & 0xffff0000u);
        }
        o[0] = make_uint4(y[0], y[1], y[2], y[3]);
        o[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
    *(uint4 *)(dst + i * 32) = o[0];
    *(uint4 *)(dst + i * 32 + 16) = o[1];
}

int bounds_lay(const drk_kv_layout *g, Lay *a, const char *who)
{
    int rc = make_lay(g, a);
    if (rc) return rc;
    if (a->D < 64 || a->D > 512 || ilog2_exact((unsigned)a->D) < 0)
        return fail(DRK_ERR_UNSUPPORTED, "%s: head_dim %d is not a power of two in [64, 512]", who, a->D);
    return DRK_OK;
}

} // namespace drk

using namespace drk;

extern "C" {

size_t drk_kv_bounds_bytes(const drk_kv_layout *g)
{
    Lay a;
    if (bounds_lay(g, &a, "kv_bounds_bytes")) return 0;
    return (bounds_exps_offset(a) + (size_t)a.L * a.NB * a.KVH + 15) & ~(size_t)15;
}

int drk_kv_bounds_update(const drk_kv_layout *g, const void *pool, const int32_t *d_tables, int table_stride, const int32_t *d_pos,
                         int pos_start, int n, int layer, int layer_count, void *bounds, void *stream)
{
    Lay a;
    int rc = bounds_lay(g, &a, "kv_bounds_update");
    if (rc) return rc;
    if (n < 0 || pos_start < 0 || table_stride < 0 || pos_start > 0x7fffffff - n)
        return fail(DRK_ERR_INVALID, "kv_bounds_update: bad argument");
    if (layer < 0 || layer_count < 0 || layer_count > a.L - layer)
        return fail(DRK_ERR_INVALID, "kv_bounds_update: layers [%d, +%d) outside [0,%d)", layer, layer_count, a.L);
    if (n == 0 || layer_count == 0) return DRK_OK;
    if (!pool || !d_tables || !bounds) return fail(DRK_ERR_INVALID, "kv_bounds_update: NULL pointer");
    if (((uintptr_t)pool | (uintptr_t)bounds) & 15u) return fail(DRK_ERR_INVALID, "kv_bounds_update: pool and bounds must be 16-byte aligned");
    BoundsArgs A;
    A.pool = (const uint8_t *)pool; A.bounds = (uint8_t *)bounds; A.tables = d_tables; A.d_pos = d_pos;
    A.exps = bounds_exps_offset(a);
    A.table_stride = table_stride; A.pos_start = pos_start; A.n = n; A.layer0 = layer;
    A.bs_div = mk_div((unsigned)a.bs);
    A.first_block = d_pos ? 0 : pos_start / a.bs;
    A.n_blocks = d_pos ? n : (pos_start + n - 1) / a.bs - A.first_block + 1;
    if (!d_pos && table_stride > 0 && A.n_blocks > table_stride - A.first_block) {      // what lies behind the table's row has no page
        if (A.first_block >= table_stride) return DRK_OK;
        A.n_blocks = table_stride - A.first_block;
    }
    const size_t units = (size_t)A.n_blocks * a.KVH * layer_count;
    if (units * (a.row_bytes / 16) > ((size_t)0x7fffffff << 8) || units > 0x7fffffffu) return fail(DRK_ERR_INVALID, "kv_bounds_update: too many blocks");
    A.units = (unsigned)units;
    const unsigned lpr = a.row_bytes / 16;
    const int lpr_shift = ilog2_exact(lpr);
    const size_t unit_bytes = (size_t)a.bs * a.row_bytes;
    const bool wide = a.bs > kBLongBlock && (units <= unit_bytes / 16 || unit_bytes >= kBLongBytes);
    const dim3 grid(wide ? (unsigned)units : (unsigned)((units * lpr + kBThreads - 1) / kBThreads));
    hipStream_t st = (hipStream_t)stream;
#define DRK_BOUNDS_LAUNCH(DT)                                                                                             \
    do {                                                                                                                  \
        if (wide) hipLaunchKernelGGL(bounds_update_long_kernel<DT>, grid, dim3(kBThreads), 0, st, a, A, lpr, lpr_shift);  \
        else hipLaunchKernelGGL(bounds_update_kernel<DT>, grid, dim3(kBThreads), 0, st, a, A, lpr, lpr_shift);            \
    } while (0)
    switch (a.dtype) {
    case DRK_F16: DRK_BOUNDS_LAUNCH(DRK_F16); break;
    case DRK_BF16: DRK_BOUNDS_LAUNCH(DRK_BF16); break;
    case DRK_INT8: DRK_BOUNDS_LAUNCH(DRK_INT8); break;
    default: DRK_BOUNDS_LAUNCH(DRK_FP8_E4M3); break;
    }
#undef DRK_BOUNDS_LAUNCH
    DRK_LAUNCH_CHECK("bounds_update_kernel");
    return DRK_OK;
}

int drk_kv_bounds_extract(const drk_kv_layout *g, void *d_dst, const void *bounds, const int32_t *d_blocks, int n_blocks, int layer,
                          int layer_count, void *stream)
{
    Lay a;
    int rc = bounds_lay(g, &a, "kv_bounds_extract");
    if (rc) return rc;
    if (n_blocks < 0) return fail(DRK_ERR_INVALID, "kv_bounds_extract: bad argument");
    if (layer < 0 || layer_count < 0 || layer_count > a.L - layer)
        return fail(DRK_ERR_INVALID, "kv_bounds_extract: layers [%d, +%d) outside [0,%d)", layer, layer_count, a.L);
    if (n_blocks == 0 || layer_count == 0) return DRK_OK;
    if (!d_dst || !bounds || !d_blocks) return fail(DRK_ERR_INVALID, "kv_bounds_extract: NULL pointer");
    if (((uintptr_t)d_dst | (uintptr_t)bounds) & 15u) return fail(DRK_ERR_INVALID, "kv_bounds_extract: d_dst and bounds must be 16-byte aligned");
    const int cps = ilog2_exact((unsigned)a.D / 8);                  // 16-code chunks of a (low, high) pair
    const size_t chunks = ((size_t)layer_count * n_blocks * a.KVH) << cps, blocks = (chunks + kBThreads - 1) / kBThreads;
    if (blocks > 0x7fffffffu) return fail(DRK_ERR_INVALID, "kv_bounds_extract: too many blocks");
    hipLaunchKernelGGL(bounds_extract_kernel, dim3((unsigned)blocks), dim3(kBThreads), 0, (hipStream_t)stream, a, (uint8_t *)d_dst,
                       (const uint8_t *)bounds, bounds_exps_offset(a), d_blocks, n_blocks, layer, chunks, cps);
    DRK_LAUNCH_CHECK("bounds_extract_kernel");
    return DRK_OK;
}

} // extern "C"
