// drk_select.hip -- which blocks of a long context a query looks at: a score of every block
// against the bounds of its keys, then the best n_keep of each (row, kv head).
//
// The score of a block is 2^(eq + e) * sum_d max(c_d low_d, c_d high_d).  With c+ = max(c, 0) and
// c- = min(c, 0) the sum is c- . low + c+ . high: a product over 2 D int8 values that the matrix
// cores form exactly (|sum| <= 127^2 D < 2^24), so the score is a whole number below 2^24 times a
// power of two -- exact in fp32, the same for every order of summation, and the selection cannot
// depend on how the work was cut.
//
// score_kernel: a wave takes 16 blocks as the rows of v_mfma_i32_16x16x64_i8 -- a block's codes lie
// as the operand wants them, 16 bytes per lane -- and 16 columns: the query heads of a kv head (padded to
// a power of two by repeating the last) of one row, or of several rows when all rows share one table.
// It leaves an ordered 32-bit key per block: 0 = not a candidate, 2^32 - 1 = always kept, otherwise
// the score's bits in an order-preserving form.
// topk_kernel: one workgroup per (row, kv head) finds the n_keep-th key by histograms of 2048 bins over
// the range the keys really span (a handful of keys remain after the first) and writes the chosen
// indices in ascending order by prefix sums of ballots: no atomics decide an order.
#include "drk_common.hpp"
#include "drk_codec.hpp"
#include "drk_bounds.hpp"

namespace drk {

constexpr uint32_t kKeyForced = 0xffffffffu;
typedef int sel_i32x4 __attribute__((ext_vector_type(4)));

struct SelArgs {
    const uint8_t *bounds, *exps;       // of the layer
    const uint8_t *q;
    const int32_t *tables, *seq_lens;
    uint32_t *keys;                     // [T][KVH][key_stride]
    int32_t *out;
    int table_stride, pos_start, T, max_seq_len, keep, sink, recent, io_dtype;
    int P, R;                           // columns per row (a power of two >= heads per kv head), rows per 16 columns
    int groups_per_wave;
    unsigned key_stride;
    Div bs_div;
};

__device__ __forceinline__ int sel_blocks_of_row(const SelArgs &A, int t)
{
    int len = A.seq_lens ? A.seq_lens[t] : A.pos_start + t + 1;
    len = min(len, A.max_seq_len);
    return len > 0 ? (int)dv((unsigned)len + A.bs_div.d - 1, A.bs_div) : 0;
}

__device__ __forceinline__ uint32_t sel_key(float s)
{
    const uint32_t u = __float_as_uint(s);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// c = rint(x * 2^-e) of 4 values as bytes, split into the negative and the positive part
__device__ __forceinline__ void sel_codes4(const float *x, float inv, uint32_t &neg, uint32_t &pos)
{
    neg = pos = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = (int)rintf(fminf(fmaxf(x[i] * inv, -127.0f), 127.0f));
        neg |= ((uint32_t)min(c, 0) & 0xffu) << (8 * i);
        pos |= ((uint32_t)max(c, 0) & 0xffu) << (8 * i);
    }
}

template <int D, int SETS>
__global__ __launch_bounds__(256) void score_kernel(Lay a, SelArgs A)
{
    constexpr int HK = D / 64, KS = 2 * HK;                  // 64-byte steps of one half / of a row of codes
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int h = blockIdx.y, GQ = a.QH / a.KVH;
    const int row0 = blockIdx.z * (A.R * SETS);
    const int first = ((int)blockIdx.x * 4 + w) * A.groups_per_wave;      // first 16-block group of this wave

    // the columns: codes of one query head each, the negative parts against the lows, the positive against the highs
    sel_i32x4 qb[SETS][KS];
    int eq[SETS], nbr[SETS], trow[SETS];
    int nbmax = 0;
#pragma unroll
    for (int s = 0; s < SETS; s++) {
        const int t = row0 + s * A.R + (A.R > 1 ? c / A.P : 0);
        trow[s] = t;
        nbr[s] = t < A.T ? sel_blocks_of_row(A, t) : 0;
        nbmax = max(nbmax, nbr[s]);
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) nbmax = max(nbmax, __shfl_xor(nbmax, off));
    if (first * 16 >= nbmax) return;
#pragma unroll
    for (int s = 0; s < SETS; s++) {
        const int t = min(trow[s], A.T - 1), head = h * GQ + min(c % A.P, GQ - 1);
        const uint8_t *qp = A.q + ((size_t)t * a.QH + head) * D * 2 + g * 32;
        float x[HK][16], amax = 0.0f;
#pragma unroll
        for (int k = 0; k < HK; k++) {
            unpack8(*(const uint4 *)(qp + k * 128), A.io_dtype, &x[k][0]);
            unpack8(*(const uint4 *)(qp + k * 128 + 16), A.io_dtype, &x[k][8]);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                x[k][i] = x[k][i] == x[k][i] ? x[k][i] : 0.0f;
                amax = fmaxf(amax, fabsf(x[k][i]));
            }
        }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        eq[s] = bounds_exponent(amax);
        const float inv = ldexpf(1.0f, -eq[s]);
#pragma unroll
        for (int k = 0; k < HK; k++) {
            uint32_t n[4], p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) sel_codes4(&x[k][4 * i], inv, n[i], p[i]);
            qb[s][k] = sel_i32x4{(int)n[0], (int)n[1], (int)n[2], (int)n[3]};
            qb[s][HK + k] = sel_i32x4{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
        }
    }
    const int32_t *tab = A.tables + (size_t)row0 * A.table_stride;

    for (int gi = first; gi < first + A.groups_per_wave && gi * 16 < nbmax; gi++) {
        const int lb = gi * 16 + c;                          // this lane's block as an operand row
        int blk = lb < nbmax ? tab[lb] : -1;
        const bool hole = blk < 0 || blk >= a.NB;
        if (hole) blk = 0;                                   // always mapped; its score is not used
        const size_t entry = (size_t)blk * a.KVH + h;
        const uint8_t *cp = A.bounds + entry * (2 * D) + g * 16;
        uint4 av[KS];
#pragma unroll
        for (int k = 0; k < KS; k++) av[k] = *(const uint4 *)(cp + k * 64);
        const int eb = hole ? 1000 : (int)(int8_t)A.exps[entry];
        int ebj[4];
#pragma unroll
        for (int j = 0; j < 4; j++) ebj[j] = __shfl(eb, 4 * g + j);
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            sel_i32x4 acc = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
            for (int k = 0; k < KS; k++)
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(sel_i32x4, av[k]), qb[s][k], acc, 0, 0, 0);
#endif
            uint32_t key[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float x = ldexpf((float)acc[j], ebj[j] == 1000 ? 0 : ebj[j] + eq[s]);
                for (int off = 1; off < A.P; off <<= 1) x = fmaxf(x, __shfl_xor(x, off));
                const int b = gi * 16 + 4 * g + j;
                key[j] = b >= nbr[s] || ebj[j] == 1000 ? 0u : (b < A.sink || b >= nbr[s] - A.recent ? kKeyForced : sel_key(x));
            }
            if (c % A.P == 0 && (A.R > 1 || c == 0) && trow[s] < A.T && (unsigned)(gi * 16 + 4 * g) < A.key_stride)
                *(uint4 *)(A.keys + ((size_t)trow[s] * a.KVH + h) * A.key_stride + gi * 16 + 4 * g) = make_uint4(key[0], key[1], key[2], key[3]);
        }
    }
}

constexpr int kSelBins = 2048;

template <int THREADS>
__global__ __launch_bounds__(THREADS) void topk_kernel(SelArgs A, int KVH)
{
    constexpr int W = THREADS / 64, NR = 8, BPT = kSelBins / THREADS, SLAB = NR * THREADS;
    __shared__ uint32_t hist[kSelBins];
    __shared__ uint32_t red[4][W];
    __shared__ uint32_t cgt[NR * W], ceq[NR * W];
    __shared__ uint32_t found[3];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int t = blockIdx.x / KVH;
    const int nb = sel_blocks_of_row(A, t);
    const uint32_t *keys = A.keys + (size_t)blockIdx.x * A.key_stride;
    int32_t *out = A.out + (size_t)blockIdx.x * A.keep;
    const int slabs = (nb + SLAB - 1) / SLAB;
    uint32_t kr[NR];
    auto load = [&](int sl) {
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int idx = sl * SLAB + i * THREADS + tid;
            kr[i] = idx < nb ? keys[idx] : 0u;
        }
    };
    // ---- how many are candidates, how many forced, which range the others span ----
    uint32_t mn = 0xffffffffu, mx = 0, nv = 0, nf = 0;
    for (int sl = 0; sl < slabs; sl++) {
        load(sl);
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const uint32_t k = kr[i];
            nf += k == kKeyForced;
            if (k != 0 && k != kKeyForced) { nv++; mn = min(mn, k); mx = max(mx, k); }
        }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        mn = min(mn, (uint32_t)__shfl_xor((int)mn, off));
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, off));
        nv += (uint32_t)__shfl_xor((int)nv, off);
        nf += (uint32_t)__shfl_xor((int)nf, off);
    }
    if (lane == 0) { red[0][w] = mn; red[1][w] = mx; red[2][w] = nv; red[3][w] = nf; }
    __syncthreads();
    nv = nf = 0;
    for (int i = 0; i < W; i++) {
        mn = min(mn, red[0][i]);
        mx = max(mx, red[1][i]);
        nv += red[2][i];
        nf += red[3][i];
    }
    // chosen: keys above thr, and the first `ties` equal to it
    uint32_t thr = 0, ties = 0;
    const uint32_t want = (uint32_t)A.keep > nf ? (uint32_t)A.keep - nf : 0u;
    if (want == 0) {
        thr = kKeyForced - 1;
    } else if (nv > want) {
        uint32_t base = mn, need = want, limit = mx - mn;                 // keys base .. base + limit are in question
        for (;;) {
            const int bits = limit ? 32 - __builtin_clz(limit) : 0, shift = bits > 11 ? bits - 11 : 0;
            for (int i = tid; i < kSelBins; i += THREADS) hist[i] = 0;
            __syncthreads();
            for (int sl = 0; sl < slabs; sl++) {
                if (slabs > 1) load(sl);
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    const uint32_t k = kr[i];
                    if (k != 0 && k != kKeyForced && k >= base && k - base <= limit) atomicAdd(&hist[(k - base) >> shift], 1u);
                }
            }
            __syncthreads();
            // counts of the bins above this thread's, from the top down
            uint32_t own[BPT], sum = 0;
#pragma unroll
            for (int i = 0; i < BPT; i++) { own[i] = hist[tid * BPT + i]; sum += own[i]; }
            uint32_t above = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t v = (uint32_t)__shfl_down((int)above, off);
                if (lane + off < 64) above += v;
            }
            if (lane == 0) red[0][w] = above;
            __syncthreads();
            above -= sum;
            for (int i = w + 1; i < W; i++) above += red[0][i];
            if (above < need && need <= above + sum) {
                uint32_t ab = above;
#pragma unroll
                for (int i = BPT - 1; i >= 0; i--) {
                    if (ab < need && need <= ab + own[i]) { found[0] = (uint32_t)(tid * BPT + i); found[1] = need - ab; found[2] = own[i]; }
                    ab += own[i];
                }
            }
            __syncthreads();
            base += found[0] << shift;
            need = found[1];
            if (found[2] == need) { thr = base - 1; break; }              // the whole bin
            if (shift == 0) { thr = base; ties = need; break; }
            limit = min((1u << shift) - 1, limit - (found[0] << shift));
            __syncthreads();
        }
    }
    // ---- the chosen ones, in ascending order ----
    uint32_t done_gt = 0, done_eq = 0;
    const uint64_t below = (1ull << lane) - 1;
    for (int sl = 0; sl < slabs; sl++) {
        if (slabs > 1) load(sl);
        __syncthreads();
        uint64_t mg[NR], me[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            mg[i] = __ballot(kr[i] > thr);
            me[i] = ties ? __ballot(kr[i] == thr) : 0ull;
            if (lane == 0) { cgt[i * W + w] = (uint32_t)__popcll(mg[i]); ceq[i * W + w] = (uint32_t)__popcll(me[i]); }
        }
        __syncthreads();
        if (w == 0) {                                                     // exclusive prefix sums of NR * W counts
            constexpr int E = (NR * W + 63) / 64;
            uint32_t sg = 0, se = 0, vg[E], ve[E];
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int x = lane * E + i;
                vg[i] = x < NR * W ? cgt[x] : 0u;
                ve[i] = x < NR * W ? ceq[x] : 0u;
                sg += vg[i];
                se += ve[i];
            }
            uint32_t ig = sg, ie = se;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t a1 = (uint32_t)__shfl_up((int)ig, off), a2 = (uint32_t)__shfl_up((int)ie, off);
                if (lane >= off) { ig += a1; ie += a2; }
            }
            if (lane == 63) { found[0] = ig; found[1] = ie; }
            ig -= sg;
            ie -= se;
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int x = lane * E + i;
                if (x < NR * W) { cgt[x] = ig; ceq[x] = ie; }
                ig += vg[i];
                ie += ve[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const uint32_t bg = done_gt + cgt[i * W + w] + (uint32_t)__popcll(mg[i] & below);
            const uint32_t be = done_eq + ceq[i * W + w] + (uint32_t)__popcll(me[i] & below);
            const bool eq = (me[i] >> lane) & 1;
            if ((((mg[i] >> lane) & 1) || (eq && be < ties))) {
                const uint32_t at = bg + min(be, ties);
                if (at < (uint32_t)A.keep) out[at] = sl * SLAB + i * THREADS + tid;
            }
        }
        done_gt += found[0];
        done_eq += found[1];
    }
    for (uint32_t i = done_gt + min(done_eq, ties) + tid; i < (uint32_t)A.keep; i += THREADS) out[i] = -1;
}

static unsigned sel_key_stride(const Lay &a, int max_seq_len)
{
    return (unsigned)(((size_t)max_seq_len + a.bs - 1) / a.bs + 3) & ~3u;
}

template <int D>
static void launch_score(const Lay &a, const SelArgs &A, int sets, dim3 grid, hipStream_t st)
{
    if constexpr (D <= 256) {
        if (sets == 4) { hipLaunchKernelGGL((score_kernel<D, 4>), grid, dim3(256), 0, st, a, A); return; }
    }
    hipLaunchKernelGGL((score_kernel<D, 1>), grid, dim3(256), 0, st, a, A);
}

} // namespace drk

using namespace drk;

extern "C" {

size_t drk_block_select_workspace_bytes(const drk_kv_layout *g, int T, int max_seq_len)
{
    Lay a;
    if (bounds_lay(g, &a, "block_select_workspace_bytes") || T < 1 || max_seq_len < 1) return 0;
    return (size_t)T * a.KVH * sel_key_stride(a, max_seq_len) * 4;
}

int drk_block_select(const drk_kv_layout *g, const void *bounds, int layer, const void *q, int io_dtype, const int32_t *d_tables,
                     int table_stride, const int32_t *d_seq_lens, int pos_start, int T, int max_seq_len, int n_keep, int n_sink,
                     int n_recent, int32_t *d_selected, void *workspace, size_t workspace_bytes, void *stream)
{
    Lay a;
    int rc = bounds_lay(g, &a, "block_select");
    if (rc) return rc;
    if (io_dtype != DRK_F16 && io_dtype != DRK_BF16) return fail(DRK_ERR_INVALID, "block_select: io_dtype must be F16 or BF16");
    if (a.QH / a.KVH > 16) return fail(DRK_ERR_UNSUPPORTED, "block_select: %d query heads per kv head, at most 16 are supported", a.QH / a.KVH);
    if (layer < 0 || layer >= a.L) return fail(DRK_ERR_INVALID, "block_select: layer %d outside [0,%d)", layer, a.L);
    if (T < 0 || max_seq_len < 0 || table_stride < 0 || pos_start < 0 || pos_start > 0x7fffffff - T)
        return fail(DRK_ERR_INVALID, "block_select: bad argument");
    if (n_keep < 1 || n_sink < 0 || n_recent < 0 || n_sink > n_keep || n_recent > n_keep - n_sink)
        return fail(DRK_ERR_INVALID, "block_select: n_sink %d + n_recent %d must be at most n_keep %d", n_sink, n_recent, n_keep);
    if (T == 0) return DRK_OK;
    if (!bounds || !q || !d_tables || !d_selected) return fail(DRK_ERR_INVALID, "block_select: NULL pointer");
    if (((uintptr_t)bounds | (uintptr_t)q | (uintptr_t)workspace) & 15u)
        return fail(DRK_ERR_INVALID, "block_select: bounds, q and the workspace must be 16-byte aligned");
    SelArgs A;
    A.key_stride = sel_key_stride(a, max_seq_len);
    const size_t need = (size_t)T * a.KVH * A.key_stride * 4;
    if (need && (!workspace || workspace_bytes < need))
        return fail(DRK_ERR_WORKSPACE, "block_select: %zu bytes of workspace, %zu needed", workspace_bytes, need);
    if ((size_t)T * a.KVH > 0x7fffffffu) return fail(DRK_ERR_INVALID, "block_select: too many rows");
    A.bounds = (const uint8_t *)bounds + (size_t)layer * a.NB * a.KVH * 2 * a.D;
    A.exps = (const uint8_t *)bounds + bounds_exps_offset(a) + (size_t)layer * a.NB * a.KVH;
    A.q = (const uint8_t *)q; A.tables = d_tables; A.seq_lens = d_seq_lens; A.keys = (uint32_t *)workspace; A.out = d_selected;
    A.table_stride = table_stride; A.pos_start = pos_start; A.T = T; A.max_seq_len = max_seq_len;
    A.keep = n_keep; A.sink = n_sink; A.recent = n_recent; A.io_dtype = io_dtype;
    A.bs_div = mk_div((unsigned)a.bs);
    A.P = 1;
    while (A.P < a.QH / a.KVH) A.P *= 2;
    A.R = table_stride == 0 ? 16 / A.P : 1;
    const int sets = table_stride == 0 && a.D <= 256 && T > A.R ? 4 : 1;
    const int n = (int)(((size_t)max_seq_len + a.bs - 1) / a.bs);
    hipStream_t st = (hipStream_t)stream;
    if (n > 0) {
        const size_t tiles = ((size_t)T + A.R * sets - 1) / (A.R * sets), groups = ((size_t)n + 15) / 16;
        if (tiles > 65535 || a.KVH > 65535) return fail(DRK_ERR_UNSUPPORTED, "block_select: %d rows are more than one launch takes", T);
        const size_t all = groups * a.KVH * tiles;                        // 16-block groups of every kv head and row tile
        A.groups_per_wave = (int)(all / 4096 < 1 ? 1 : (all / 4096 > 16 ? 16 : all / 4096));
        const dim3 grid((unsigned)((groups + 4 * A.groups_per_wave - 1) / (4 * A.groups_per_wave)), a.KVH, (unsigned)tiles);
        switch (a.D) {
        case 64: launch_score<64>(a, A, sets, grid, st); break;
        case 128: launch_score<128>(a, A, sets, grid, st); break;
        case 256: launch_score<256>(a, A, sets, grid, st); break;
        default: launch_score<512>(a, A, sets, grid, st); break;
        }
        DRK_LAUNCH_CHECK("score_kernel");
    }
    if (n > 2048) hipLaunchKernelGGL((topk_kernel<1024>), dim3(T * a.KVH), dim3(1024), 0, st, A, a.KVH);
    else hipLaunchKernelGGL((topk_kernel<256>), dim3(T * a.KVH), dim3(256), 0, st, A, a.KVH);
    DRK_LAUNCH_CHECK("topk_kernel");
    return DRK_OK;
}

} // extern "C"
