// drk_select.hip -- which blocks of a long context a query looks at: a score of every block
// against the bounds of its keys, then the best n_keep of each (row, kv head).
//
// The score of a block is 2^(eq + e) * sum_d max(c_d low_d, c_d high_d).  With c+ = max(c, 0) and
// c- = min(c, 0) the sum is c- . low + c+ . high: a product over 2 D int8 values that the matrix
// cores form exactly (|sum| <= 127^2 D < 2^24), so the score is a whole number below 2^24 times a
// power of two -- exact in fp32, the same for every order of summation, and the selection cannot
// depend on how the work was cut.
//
// The score kernels form v_mfma_i32_16x16x64_i8 products of 16 query heads (rows) with 16 blocks (columns): a
// block's codes lie as the operand wants them, 16 bytes per lane, and the result has a block per lane and
// four heads in its registers, so the largest score over a kv head's heads is mostly formed in a lane.  They
// leave an ordered 32-bit key per block: 0 = not a candidate, 2^32 - 1 = always kept, otherwise the score's
// bits in an order-preserving form.
//   score_kernel: a wave scores its own blocks for one set of 16 heads -- branches, whose blocks nobody else
//   reads.  Bound by the bytes of the bounds: 16 branches x up to 64k (101 MB) 20 us, 5.1 TB/s and about 5 us of launch, length,
//   table and first codes; one branch x 32k 4 us.
//   score_tile_kernel: rows of one table; 8 waves x 2 sets of heads meet the same blocks, which pass through LDS.  512 rows x
//   24 heads x 1970 blocks of head_dim 256: 29 us, 0.84 POP/s (1.13 with the rows that fill up an operand: 8 for 6 heads):
//   per 32 blocks and wave 32 products (512 clocks), 16 LDS reads and 123 vector instructions (about as long each), which
//   two waves per SIMD overlap by half; another 5 us are the queries' conversion.
// topk_kernel: one workgroup per (row, kv head) finds the n_keep-th key: a histogram over the range the keys
// really span leaves a handful in one bin, which every wave then settles by itself with ballots; the chosen
// indices are written in ascending order by prefix sums of ballots.  No atomic decides an order.  Bound by its dozen exchanges:
// 8 rows of 2048 keys 5 us, 128 of up to 4096 6.8, 2048 of 1970 13.
#include "drk_common.hpp"
#include "drk_codec.hpp"
#include "drk_bounds.hpp"

#include <type_traits>

namespace drk {

constexpr uint32_t kKeyForced = 0xffffffffu;
// Contexts of few blocks are scored and selected by one workgroup per (row, kv head) in one launch: a second launch costs
// about 3 us, one workgroup reads some 60 GB/s.  A branch of 8 kv heads x 128: 250 blocks 6.9 us; 500 blocks 8.2 where the
// two kernels take 10.1; 750 blocks 9.5 and 10.1; 1000 blocks 10.6 and 9.7.
constexpr size_t kSelFusedBytes = 200 << 10;   // codes of the context per kv head, with few rows
constexpr int kSelFusedRows = 256;             // (row, kv head) pairs that keep every CU busy by themselves
constexpr int kSelFused = 1024;                // blocks, the most that kernel takes
constexpr int kSelShort = 128;                 // blocks up to which chunks take it too, and fewer threads do
constexpr int kSelWaveGroups = 4;              // 16-block groups of a wave of score_kernel: 64 table entries
constexpr size_t kSelWaves = 4096;             // waves that a decode step's scores are spread over
constexpr unsigned kSelTileWgs = 256;          // CUs that a chunk's workgroups are spread over
constexpr unsigned kSelTileStart = 6;          // what such a workgroup spends on its queries, counted in groups
typedef int sel_i32x4 __attribute__((ext_vector_type(4)));

struct SelArgs {
    const uint8_t *bounds, *exps;       // of the layer
    const uint8_t *q;
    const int32_t *tables, *seq_lens;
    uint32_t *keys;                     // [T][KVH][key_stride]
    int32_t *out;
    int table_stride, pos_start, T, max_seq_len, keep, sink, recent, io_dtype;
    int P, R;                           // operand rows per query row (a power of two >= heads per kv head), query rows per 16
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
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ float sel_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// ---- query heads as an operand ----------------------------------------------------------------------
// Four codes (the low bytes of u = 1.5 * 2^23 + c) as one dword, split into its negative and its positive bytes: the byte
// above a code is 0xff where the code is negative and 0 elsewhere.
__device__ __forceinline__ void sel_split4(const uint32_t (&u)[4], uint32_t &neg, uint32_t &pos)
{
    const uint32_t a = s_perm(u[1], u[0], 0x05010400u), b = s_perm(u[3], u[2], 0x05010400u);
    const uint32_t c = s_perm(b, a, 0x05040100u), mask = s_perm(b, a, 0x07060302u);
    neg = c & mask;
    pos = c & ~mask;
}

// x 2^-e rounded to the nearest whole number, as sel_split4 takes it, of the HK * 16 dims of a lane
template <int HK, bool BF16>
__device__ __forceinline__ void sel_codes(const uint4 (&raw)[HK][2], float inv, sel_i32x4 *qa)
{
#pragma unroll
    for (int k = 0; k < HK; k++) {
        uint32_t n[4], p[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint4 &r = raw[k][j >> 1];
            const uint32_t w[2] = {j & 1 ? r.z : r.x, j & 1 ? r.w : r.y};
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float x;
                if constexpr (BF16) x = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
                else x = (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]));
                u[i] = __float_as_uint(__builtin_fmaf(x, inv, 12582912.0f));
            }
            sel_split4(u, n[j], p[j]);
        }
        qa[k] = sel_i32x4{(int)n[0], (int)n[1], (int)n[2], (int)n[3]};
        qa[HK + k] = sel_i32x4{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
    }
}

// Codes c = rint(q 2^-eq) of one head row; lane (c, g) holds dims 64 k + 16 g .. + 15: the negative parts meet the
// lows (first D / 64 steps), the positive parts the highs.  Adding 1.5 * 2^23 to x * 2^-e in one fused operation rounds to
// the nearest whole number, ties to even, and leaves the code as the low byte: the product is exact and at most 127.
// Rows with a NaN, or beyond the exponents' range, take the long way.
template <int D>
__device__ __forceinline__ int sel_query(const uint8_t *row, int g, int io_dtype, sel_i32x4 *qa)
{
    constexpr int HK = D / 64;
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    uint4 raw[HK][2];
#pragma unroll
    for (int k = 0; k < HK; k++) {
        raw[k][0] = *(const uint4 *)(row + k * 128 + g * 32);
        raw[k][1] = *(const uint4 *)(row + k * 128 + g * 32 + 16);
    }
    u16x2 m2 = {0, 0};                                                          // magnitudes order like their bits
#pragma unroll
    for (int k = 0; k < HK; k++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t w[4] = {raw[k][j].x, raw[k][j].y, raw[k][j].z, raw[k][j].w};
#pragma unroll
            for (int i = 0; i < 4; i++) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        }
    int m = max((int)m2.x, (int)m2.y);
    m = max(m, __shfl_xor(m, 16));
    m = max(m, __shfl_xor(m, 32));
    int e = bounds_exponent(elem16_to_f((uint16_t)m, io_dtype));
    if (__ballot(m > (io_dtype == DRK_BF16 ? 0x7f80 : 0x7c00) || e == 40) == 0) {
        if (io_dtype == DRK_BF16) sel_codes<HK, true>(raw, sel_pow2(-e), qa);
        else sel_codes<HK, false>(raw, sel_pow2(-e), qa);
        return e;
    }
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < HK; k++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float x[8];
            unpack8(raw[k][j], io_dtype, x);
#pragma unroll
            for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[i]));        // NaN is passed over
        }
    amax = fmaxf(amax, __shfl_xor(amax, 16));
    amax = fmaxf(amax, __shfl_xor(amax, 32));
    e = bounds_exponent(amax);
    const float inv = sel_pow2(-e);
#pragma unroll
    for (int k = 0; k < HK; k++) {
        uint32_t n[4], p[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x[8];
            uint32_t u[4];
            unpack8(raw[k][j >> 1], io_dtype, x);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float y = x[4 * (j & 1) + i] * inv;
                u[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(y == y ? y : 0.0f, -127.0f), 127.0f), 12582912.0f));
            }
            sel_split4(u, n[j], p[j]);
        }
        qa[k] = sel_i32x4{(int)n[0], (int)n[1], (int)n[2], (int)n[3]};
        qa[HK + k] = sel_i32x4{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
    }
    return e;
}

// Heads 4g + j of one product against block c: the key of the largest score over the P heads of a row (P = 4, 8 or 16), in
// every lane of the row.  qm = 2^eq of the heads, bm = 2^e of the block.  A row's other heads are 16 (and 32) lanes
// away: the two results of a swap with itself are the two sides.
template <int P>
__device__ __forceinline__ uint32_t sel_row_key(const sel_i32x4 &acc, const float *qm, float bm)
{
    const float x = fmaxf(fmaxf((float)acc[0] * qm[0], (float)acc[1] * qm[1]), fmaxf((float)acc[2] * qm[2], (float)acc[3] * qm[3]));
    uint32_t k = sel_key(x * bm);
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (P >= 8) {
        const auto s = __builtin_amdgcn_permlane16_swap(k, k, false, false);
        k = max((uint32_t)s[0], (uint32_t)s[1]);
    }
    if constexpr (P >= 16) {
        const auto s = __builtin_amdgcn_permlane32_swap(k, k, false, false);
        k = max((uint32_t)s[0], (uint32_t)s[1]);
    }
#endif
    return k;
}
__device__ __forceinline__ uint32_t sel_row_key(const sel_i32x4 &acc, const float *qm, int P, float bm)
{
    return P == 4 ? sel_row_key<4>(acc, qm, bm) : (P == 8 ? sel_row_key<8>(acc, qm, bm) : sel_row_key<16>(acc, qm, bm));
}

constexpr int kNoBlock = 1000;          // in place of the exponent of a block without a page

__device__ __forceinline__ uint32_t sel_key_of(const SelArgs &A, uint32_t scored, int b, int nb, int e)
{
    const bool forced = (b < A.sink) | (b >= nb - A.recent), none = (b >= nb) | (e == kNoBlock);
    return none ? 0u : (forced ? kKeyForced : scored);
}

// The codes of 16 blocks on their way to a wave's operands.  An operand's neighbouring lanes hold neighbouring blocks, and lanes
// 16 apart the same block's chunks: read like that, every lane is an access of its own (51 per load, 9.4 M of them for
// 16 branches x 64k: the score kernel's time).  So the wave reads whole blocks, lane after lane, and exchanges the
// chunks through LDS, chunk x of block c in place x ^ swap(c), which puts 16 neighbouring lanes on 16 different
// 16-byte places of the 256 that the banks hold.  The wave's own region: no barrier.
__device__ __forceinline__ int sel_swap(int D, int c) { return D == 64 ? c >> 1 : c; }
// the entry (block * KVH + head) of block c of the group lies behind the table entry in lane base + c
template <int D>
__device__ __forceinline__ void sel_fetch(sel_i32x4 (&v)[D / 32], const uint8_t *bounds, const Lay &a, int h, int ahead, int base, int lane)
{
    constexpr int CH = D / 8;                                // 16-byte chunks of a block
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
        const int x = i * 64 + lane, blk = __shfl(ahead, base + x / CH);
        const size_t entry = (size_t)((unsigned)blk < (unsigned)a.NB ? blk : 0) * a.KVH + h;   // block 0 is always mapped; its score is not used
        v[i] = *(const sel_i32x4 *)(bounds + entry * (2 * D) + (x & (CH - 1)) * 16);
    }
}
template <int D>
__device__ __forceinline__ void sel_stage(sel_i32x4 *lds, const sel_i32x4 (&v)[D / 32], int lane)
{
    constexpr int CH = D / 8;
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
        const int x = i * 64 + lane, c = x / CH;
        lds[c * CH + ((x & (CH - 1)) ^ sel_swap(D, c))] = v[i];
    }
}
template <int D>
__device__ __forceinline__ sel_i32x4 sel_operand(const sel_i32x4 *lds, int k, int g, int c)
{
    return lds[c * (D / 8) + ((k * 4 + g) ^ sel_swap(D, c))];
}
// what other lanes of the wave wrote to LDS before is there, what they read has been read
__device__ __forceinline__ void sel_wave_order()
{
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#endif
}

// One set of 16 heads per wave: a branch's row (R = 1), or R = 16 / P rows of one table.  A wave takes at most
// kSelWaveGroups groups of 16 blocks: their table entries are its lanes' one load.
template <int D>
__global__ __launch_bounds__(256) void score_kernel(Lay a, SelArgs A)
{
    constexpr int KS = D / 32;
    __shared__ sel_i32x4 codes[4][16 * D / 8];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int h = blockIdx.x, GQ = a.QH / a.KVH;           // kv heads vary fastest: a block's codes of all heads lie together
    const int row0 = blockIdx.z * A.R;
    const int first = ((int)blockIdx.y * 4 + w) * A.groups_per_wave;
    const int32_t *tab = A.tables + (size_t)row0 * A.table_stride;
    // the row of this lane's results (heads 4g .. 4g + 3), and the wave's longest
    const int row = A.R > 1 ? row0 + 4 * g / A.P : row0;
    const int nbr = row < A.T ? sel_blocks_of_row(A, row) : 0;
    const int nbmax = max(max(__shfl(nbr, 0), __shfl(nbr, 16)), max(__shfl(nbr, 32), __shfl(nbr, 48)));
    if (first * 16 >= nbmax) return;
    const int ahead = first * 16 + lane < nbmax ? tab[first * 16 + lane] : -1;  // the table entries of all its groups

    const int qrow = min(A.R > 1 ? row0 + c / A.P : row0, A.T - 1);
    sel_i32x4 qa[KS];
    const int eq = sel_query<D>(A.q + ((size_t)qrow * a.QH + h * GQ + min(c & (A.P - 1), GQ - 1)) * D * 2, g, A.io_dtype, qa);
    float qm[4];
#pragma unroll
    for (int j = 0; j < 4; j++) qm[j] = sel_pow2(__shfl(eq, 4 * g + j));

    sel_i32x4 bv[KS];
    int eb = 0;
    auto fetch = [&](int i) {                                                   // group first + i
        sel_fetch<D>(bv, A.bounds, a, h, ahead, i * 16, lane);
        const int blk = __shfl(ahead, i * 16 + c);
        eb = (unsigned)blk < (unsigned)a.NB ? (int)(int8_t)A.exps[(size_t)blk * a.KVH + h] : kNoBlock;
    };
    fetch(0);
    const int n = min(A.groups_per_wave, (nbmax + 15) / 16 - first);
    for (int i = 0; i < n; i++) {
        sel_wave_order();
        sel_stage<D>(codes[w], bv, lane);
        sel_wave_order();
        const int e = eb;
        if (i + 1 < n) fetch(i + 1);
        sel_i32x4 acc = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int k = 0; k < KS; k++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[k], sel_operand<D>(codes[w], k, g, c), acc, 0, 0, 0);
#endif
        const uint32_t x = sel_row_key(acc, qm, A.P, e == kNoBlock ? 0.0f : sel_pow2(e));
        const int b = (first + i) * 16 + c;
        if ((A.R > 1 ? ((4 * g) & (A.P - 1)) == 0 : g == 0) && row < A.T && (unsigned)b < A.key_stride)
            A.keys[((size_t)row * a.KVH + h) * A.key_stride + b] = sel_key_of(A, x, b, nbr, e);
    }
}

// Rows of one table.  A workgroup's 8 waves hold SETS sets of 16 heads each (8 SETS R rows together) and walk the same
// blocks, 32 at a time, whose codes the workgroup stages in LDS, two buffers by turns, requested two steps ahead: every
// byte of the bounds is read once per 8 SETS R rows.
template <int D, int SETS, int P>
__global__ __launch_bounds__(512) void score_tile_kernel(Lay a, SelArgs A)
{
    constexpr int KS = D / 32, CH = 2 * D / 16;              // 16-byte chunks of a block's codes
    constexpr int R = 16 / P;                                // rows per set
    constexpr int PITCH = 2 * D + 16, G = 2, PER = (16 * G * CH + 511) / 512;
    static_assert(512 % CH == 0, "a thread's chunks are the same one of several blocks");
    __shared__ __align__(16) uint8_t b_lds[2][16 * G * PITCH];
    __shared__ int e_lds[2][16 * G];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int h = blockIdx.x, GQ = a.QH / a.KVH;
    const int row0 = (int)blockIdx.z * (8 * SETS * R), wrow0 = row0 + w * SETS * R;
    const int first = (int)blockIdx.y * A.groups_per_wave;   // 16-block groups; a workgroup takes an even number
    const int last_row = min(row0 + 8 * SETS * R, A.T) - 1;
    // lengths may be any where they are given: the workgroup walks to its longest row
    int nbmax = 0;
    for (int r = row0 + lane; r <= last_row; r += 64) nbmax = max(nbmax, sel_blocks_of_row(A, r));
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) nbmax = max(nbmax, __shfl_xor(nbmax, off));
    if (first * 16 >= nbmax) return;
    const int n = (min(A.groups_per_wave, (nbmax + 15) / 16 - first) + G - 1) / G;         // steps

    // Thread (r0, ch) brings chunk ch of blocks r0, r0 + 512 / CH, .. of a step, requested two steps ahead, by table entries
    // requested two steps before that.  Even and odd steps have registers of their own and every request is made by every thread
    // (clamped instead of skipped): loads and stores are counted in order, so that a wait for a step's codes lets what
    // was requested after them travel on -- unless the compiler has to reckon with requests that were not made.
    const int r0 = (int)threadIdx.x / CH, ch = (int)threadIdx.x - r0 * CH;
    sel_i32x4 st[2][PER];
    int es[2][PER], ahead[2][PER];
    bool hole[2][PER];
    auto page = [&](int q, int i) {
#pragma unroll
        for (int u = 0; u < PER; u++) ahead[q][u] = A.tables[min((first + i * G) * 16 + r0 + u * (512 / CH), nbmax - 1)];
    };
    auto fetch = [&](int q, int i) {
#pragma unroll
        for (int u = 0; u < PER; u++) {
            hole[q][u] = (unsigned)ahead[q][u] >= (unsigned)a.NB || (first + i * G) * 16 + r0 + u * (512 / CH) >= nbmax;
            const size_t entry = (size_t)(hole[q][u] ? 0 : ahead[q][u]) * a.KVH + h;     // block 0 is always mapped
            st[q][u] = *(const sel_i32x4 *)(A.bounds + entry * (2 * D) + ch * 16);
            es[q][u] = (int)(int8_t)A.exps[entry];
        }
    };
    auto stage = [&](int q) {
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int r = r0 + u * (512 / CH);
            if (r < 16 * G) *(sel_i32x4 *)(b_lds[q] + r * PITCH + ch * 16) = st[q][u];
            if (r < 16 * G && ch == 0) e_lds[q][r] = hole[q][u] ? kNoBlock : es[q][u];
        }
    };
    page(0, 0);
    page(1, 1);
    fetch(0, 0);
    page(0, 2);
    sel_i32x4 qa[SETS][KS];
    float qm[SETS][4];
    int nbr[SETS];
    unsigned ko[SETS];                                       // keys of the lane's rows, counted from the workgroup's first row
    bool on[SETS];
    uint32_t *const kbase = A.keys + ((size_t)row0 * a.KVH + h) * A.key_stride;
    int nbmin = 0x7fffffff;
#pragma unroll
    for (int s = 0; s < SETS; s++) {
        const int qrow = min(wrow0 + s * R + c / P, A.T - 1);
        const int eq = sel_query<D>(A.q + ((size_t)qrow * a.QH + h * GQ + min(c & (P - 1), GQ - 1)) * D * 2, g, A.io_dtype, qa[s]);
#pragma unroll
        for (int j = 0; j < 4; j++) qm[s][j] = sel_pow2(__shfl(eq, 4 * g + j));
        const int row = wrow0 + s * R + 4 * g / P;
        nbr[s] = row < A.T ? sel_blocks_of_row(A, row) : 0;
        on[s] = ((4 * g) & (P - 1)) == 0 && row < A.T;
        ko[s] = (unsigned)(row - row0) * (unsigned)a.KVH * A.key_stride;
        nbmin = min(nbmin, nbr[s]);
    }
#pragma unroll
    for (int off = 16; off < 64; off <<= 1) nbmin = min(nbmin, __shfl_xor(nbmin, off));
    const int scored_end = __builtin_amdgcn_readfirstlane(nbmin) - A.recent;    // from the first blocks to here every row only scores
    // a key that is not to be stored gets an offset beyond the buffer, which the store drops: see above, no store is skipped
    const __amdgpu_buffer_rsrc_t krsrc = __builtin_amdgcn_make_buffer_rsrc(kbase, 0, (int)(64u * (unsigned)a.KVH * A.key_stride * 4), 0x00027000);
    fetch(1, 1);
    page(1, 3);
    stage(0);
    __syncthreads();
    auto step = [&](auto parity, int i) {
        constexpr int q = decltype(parity)::value;
        fetch(q, i + 2);
        page(q, i + 4);
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_sched_barrier(0);
#endif
        const uint8_t *buf = b_lds[q];
        uint4 bv[G][KS];
#pragma unroll
        for (int x = 0; x < G; x++)
#pragma unroll
            for (int k = 0; k < KS; k++) bv[x][k] = *(const uint4 *)(buf + (x * 16 + c) * PITCH + k * 64 + g * 16);
        // G * SETS chains of products side by side, then what becomes of them
        sel_i32x4 acc[G][SETS];
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int x = 0; x < G; x++)
#pragma unroll
                for (int s = 0; s < SETS; s++) {
                    if (k == 0) acc[x][s] = sel_i32x4{0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
                    acc[x][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[s][k], __builtin_bit_cast(sel_i32x4, bv[x][k]), acc[x][s], 0, 0, 0);
#endif
                }
#pragma unroll
        for (int x = 0; x < G; x++) {
            const int e = e_lds[q][x * 16 + c], b0 = (first + i * G + x) * 16, b = b0 + c;
            const bool hole = e == kNoBlock, inner = b0 >= A.sink && b0 + 16 <= scored_end;
            const float bm = hole ? 0.0f : sel_pow2(e);
            uint32_t key[SETS];
#pragma unroll
            for (int s = 0; s < SETS; s++) key[s] = hole ? 0u : sel_row_key<P>(acc[x][s], qm[s], bm);
            if (!inner) {                                    // the same for the whole wave
#pragma unroll
                for (int s = 0; s < SETS; s++) {
                    const bool forced = (b < A.sink) | (b >= nbr[s] - A.recent);
                    key[s] = (b >= nbr[s] || hole) ? 0u : (forced ? kKeyForced : key[s]);
                }
            }
#pragma unroll
            for (int s = 0; s < SETS; s++)
                __builtin_amdgcn_raw_buffer_store_b32(key[s], krsrc, (on[s] & ((unsigned)b < A.key_stride)) ? (int)((ko[s] + (unsigned)b) * 4) : -1, 0, 0);
        }
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_sched_barrier(0);
#endif
        stage(1 - q);
        __syncthreads();
    };
    for (int i = 0; i < n; i += 2) {                         // a step too many meets holes
        step(std::integral_constant<int, 0>(), i);
        step(std::integral_constant<int, 1>(), i + 1);
    }
}

// ---- the n_keep best keys ------------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sel_dpp(uint32_t v)                     // 0 where the source lane does not exist
{
#if defined(__HIP_DEVICE_COMPILE__)
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
#else
    return v;
#endif
}
// inclusive prefix sum over the wave: row shifts by 1, 2, 4, 8, then lane 15 of a row into the next, lane 31 into the rest
__device__ __forceinline__ uint32_t sel_scan(uint32_t v)
{
    v += sel_dpp<0x111, 0xf>(v);
    v += sel_dpp<0x112, 0xf>(v);
    v += sel_dpp<0x114, 0xf>(v);
    v += sel_dpp<0x118, 0xf>(v);
    v += sel_dpp<0x142, 0xa>(v);
    v += sel_dpp<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint32_t sel_lane(uint32_t v, int l)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return (uint32_t)__builtin_amdgcn_readlane((int)v, l);
#else
    (void)l;
    return v;
#endif
}
__device__ __forceinline__ uint32_t sel_wave_max(uint32_t v)                // the largest, in every lane
{
    v = max(v, sel_dpp<0xB1, 0xf>(v));
    v = max(v, sel_dpp<0x4E, 0xf>(v));
    v = max(v, sel_dpp<0x141, 0xf>(v));
    v = max(v, sel_dpp<0x140, 0xf>(v));
    return max(max(sel_lane(v, 0), sel_lane(v, 16)), max(sel_lane(v, 32), sel_lane(v, 48)));
}

constexpr uint32_t kSelList = 64;       // keys of the deciding bin that a wave settles by itself

template <int THREADS> struct TopkLds {
    static constexpr int W = THREADS / 64, BIN_BITS = THREADS >= 1024 ? 11 : 10, BINS = 1 << BIN_BITS;
    uint32_t hist[BINS], red[4][W], above_w[W], chosen_w[2][W], found[3], list[kSelList], list_n;
};

// The workgroup's part of one (row, kv head).  Keys come in slabs of NR * THREADS: fetch(slab, kr) leaves NR keys per thread,
// key i of lane l of wave w being block slab * SLAB + (w * NR + i) * 64 + l (0 from the row's end on) -- a wave's keys are
// neighbours, so that only one count per wave is exchanged when the chosen ones are written.  The first slab's
// keys are in kr already; MULTI: there may be more.  (The code runs once per workgroup, so its length is time: about
// 10 KB of it, with the refetching of slabs in it and the waves' figures added up one by one, cost 6.2 us at 2048 keys.)
template <int THREADS, int NR, bool MULTI, typename F>
__device__ __forceinline__ void topk_run(TopkLds<THREADS> &S, uint32_t (&kr)[NR], int nb, int keep, int32_t *out, F fetch)
{
    using L = TopkLds<THREADS>;
    constexpr int W = L::W, BIN_BITS = L::BIN_BITS, BINS = L::BINS, BPT = BINS / THREADS, SLAB = NR * THREADS;
    static_assert(BPT * THREADS == BINS, "every thread owns whole bins");
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slabs = MULTI ? (nb + SLAB - 1) / SLAB : 1;
    auto scored = [](uint32_t k) { return k - 1u < kKeyForced - 1u; };      // neither 0 nor kKeyForced
    auto before = [&](const uint32_t *x) {                                  // what the waves before this one left
        const uint32_t s = sel_scan(lane < W ? x[lane] : 0u);
        return w ? sel_lane(s, w - 1) : 0u;
    };
    // ---- how many are candidates, how many forced, which range the others span ----
    uint32_t mnc = 0, mx = 0, nv = 0, nf = 0;                           // mnc: the complement of the smallest
    for (int sl = 0; sl < slabs; sl++) {
        if (MULTI && sl > 0) fetch(sl, kr);
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const uint32_t k = kr[i];
            nf += (uint32_t)__popcll(__ballot(k == kKeyForced));
            nv += (uint32_t)__popcll(__ballot(scored(k)));
            if (scored(k)) { mnc = max(mnc, ~k); mx = max(mx, k); }
        }
    }
    mnc = sel_wave_max(mnc);
    mx = sel_wave_max(mx);
    if (lane == 0) { S.red[0][w] = mnc; S.red[1][w] = mx; S.red[2][w] = nv; S.red[3][w] = nf; }
    for (int i = tid; i < BINS; i += THREADS) S.hist[i] = 0;
    if (tid == 0) S.list_n = 0;
    __syncthreads();
    mnc = sel_wave_max(lane < W ? S.red[0][lane] : 0u);
    mx = sel_wave_max(lane < W ? S.red[1][lane] : 0u);
    nv = sel_lane(sel_scan(lane < W ? S.red[2][lane] : 0u), W - 1);
    nf = sel_lane(sel_scan(lane < W ? S.red[3][lane] : 0u), W - 1);
    // chosen: keys above thr, and -- where not all of them fit -- the first `ties` equal to it
    uint32_t thr = 0, ties = 0;
    const uint32_t want = (uint32_t)keep > nf ? (uint32_t)keep - nf : 0u;
    if (want == 0) {
        thr = kKeyForced - 1;
    } else if (nv > want) {
        uint32_t base = ~mnc, need = want, limit = mx - base;               // keys base .. base + limit are in question
        for (;;) {
            const int bits = limit ? 32 - __builtin_clz(limit) : 0, shift = bits > BIN_BITS ? bits - BIN_BITS : 0;
            auto in_range = [&](uint32_t k) { return scored(k) && k >= base && k - base <= limit; };
            for (int sl = 0; sl < slabs; sl++) {
                if (MULTI) fetch(sl, kr);
#pragma unroll
                for (int i = 0; i < NR; i++)
                    if (in_range(kr[i])) atomicAdd(&S.hist[(kr[i] - base) >> shift], 1u);
            }
            __syncthreads();
            // thread tid owns BPT bins, counted from the top
            uint32_t own[BPT], sum = 0;
#pragma unroll
            for (int i = 0; i < BPT; i++) { own[i] = S.hist[BINS - 1 - (tid * BPT + i)]; sum += own[i]; }
            const uint32_t incl = sel_scan(sum);
            if (lane == 63) S.above_w[w] = incl;
            __syncthreads();
            uint32_t above = incl - sum + before(S.above_w);
            if (above < need && need <= above + sum) {
#pragma unroll
                for (int i = 0; i < BPT; i++) {
                    if (above < need && need <= above + own[i]) {
                        S.found[0] = (uint32_t)(BINS - 1 - (tid * BPT + i));
                        S.found[1] = need - above;
                        S.found[2] = own[i];
                    }
                    above += own[i];
                }
            }
            __syncthreads();
            const uint32_t bin = S.found[0], in_bin = S.found[2];
            need = S.found[1];
            base += bin << shift;
            if (in_bin == need) { thr = base - 1; break; }                  // the whole bin
            if (shift == 0) { thr = base; ties = need; break; }
            limit = min((1u << shift) - 1, limit - (bin << shift));
            if (in_bin <= kSelList) {
                // few are left: every wave settles them by itself, counting for each how many are larger
                for (int sl = 0; sl < slabs; sl++) {
                    if (MULTI) fetch(sl, kr);
                    uint32_t hits = 0;
#pragma unroll
                    for (int i = 0; i < NR; i++) hits |= in_range(kr[i]) ? 1u << i : 0u;
                    if (hits) {
                        uint32_t at = atomicAdd(&S.list_n, (uint32_t)__popc(hits));
#pragma unroll
                        for (int i = 0; i < NR; i++)
                            if (hits >> i & 1) S.list[at++] = kr[i] - base;
                    }
                }
                __syncthreads();
                const uint32_t mine = S.list[min((uint32_t)lane, in_bin - 1)];
                uint32_t larger = 0, equal = 0;
                for (uint32_t i = 0; i < in_bin; i++) {
                    const uint32_t o = sel_lane(mine, (int)i);
                    larger += o > mine;
                    equal += o == mine;
                }
                const uint64_t it = __ballot(larger < need && need <= larger + equal);        // lanes that hold the need-th largest
                const int at = __builtin_ctzll(it);
                thr = base + sel_lane(mine, at);
                ties = need - sel_lane(larger, at);
                if (ties == sel_lane(equal, at)) { thr--; ties = 0; }
                break;
            }
            for (int i = tid; i < BINS; i += THREADS) S.hist[i] = 0;
            __syncthreads();
        }
    }
    // ---- the chosen ones, in ascending order ----
    auto lower = [](uint64_t m) {                                           // set bits below this lane's
#if defined(__HIP_DEVICE_COMPILE__)
        return (uint32_t)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
#else
        return (uint32_t)m;
#endif
    };
    uint32_t done_gt = 0, done_eq = 0;
    for (int sl = 0; sl < slabs; sl++) {
        if (MULTI) fetch(sl, kr);
        if (MULTI && sl > 0) __syncthreads();                                        // the counts of the slab before have been read
        uint32_t cg = 0, ce = 0;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            cg += (uint32_t)__popcll(__ballot(kr[i] > thr));
            if (ties) ce += (uint32_t)__popcll(__ballot(kr[i] == thr));
        }
        if (lane == 0) { S.chosen_w[0][w] = cg; S.chosen_w[1][w] = ce; }
        __syncthreads();
        const uint32_t sg = sel_scan(lane < W ? S.chosen_w[0][lane] : 0u), se = sel_scan(lane < W ? S.chosen_w[1][lane] : 0u);
        uint32_t bg = done_gt + (w ? sel_lane(sg, w - 1) : 0u), be = done_eq + (w ? sel_lane(se, w - 1) : 0u);
        done_gt += sel_lane(sg, W - 1);
        done_eq += sel_lane(se, W - 1);
        const int b0 = sl * SLAB + w * NR * 64 + lane;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const uint64_t mg = __ballot(kr[i] > thr);
            uint32_t at = bg + lower(mg);
            bool take = kr[i] > thr;
            if (ties) {
                const uint64_t me = __ballot(kr[i] == thr);
                const uint32_t rank = be + lower(me);
                take = take || (kr[i] == thr && rank < ties);
                at += min(rank, ties);
                be += (uint32_t)__popcll(me);
            }
            if (take && at < (uint32_t)keep) out[at] = b0 + i * 64;
            bg += (uint32_t)__popcll(mg);
        }
    }
    for (uint32_t i = done_gt + min(done_eq, ties) + tid; i < (uint32_t)keep; i += THREADS) out[i] = -1;
}

template <int THREADS, int NR, bool MULTI>
__global__ __launch_bounds__(THREADS) void topk_kernel(SelArgs A, int KVH)
{
    constexpr int SLAB = NR * THREADS;
    __shared__ TopkLds<THREADS> S;
    const int tid = threadIdx.x;
    const uint32_t *keys = A.keys + (size_t)blockIdx.x * A.key_stride;
    uint32_t kr[NR];
    const int b0 = (tid >> 6) * NR * 64 + (tid & 63);
    // the first slab is requested before the row's length is known, and cut afterwards
#pragma unroll
    for (int i = 0; i < NR; i++) kr[i] = (unsigned)(b0 + i * 64) < A.key_stride ? keys[b0 + i * 64] : 0u;
    const int nb = sel_blocks_of_row(A, blockIdx.x / KVH);
#pragma unroll
    for (int i = 0; i < NR; i++) kr[i] = b0 + i * 64 < nb ? kr[i] : 0u;
    topk_run<THREADS, NR, MULTI>(S, kr, nb, A.keep, A.out + (size_t)blockIdx.x * A.keep, [&](int sl, uint32_t (&k)[NR]) {
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int idx = sl * SLAB + b0 + i * 64;
            k[i] = idx < nb ? keys[idx] : 0u;
        }
    });
}

// Scores and selection of one (row, kv head) in one workgroup, for contexts of few blocks: the keys stay in LDS.  A wave
// asks for the table entries, then for the codes, of up to four groups at once, so that the kernel is three round
// trips to memory (length, table, codes) and the selection.
template <int D, int THREADS, int BLOCKS>
__global__ __launch_bounds__(THREADS) void select_kernel(Lay a, SelArgs A)
{
    constexpr int W = THREADS / 64, NR = BLOCKS / THREADS > 0 ? BLOCKS / THREADS : 1, KS = D / 32, GPW = BLOCKS / 16 / W;
    constexpr int G = GPW < 4 ? GPW : 4;
    static_assert(GPW * 16 * W == BLOCKS && GPW % G == 0, "whole rounds of groups");
    __shared__ TopkLds<THREADS> S;
    __shared__ uint32_t key_lds[BLOCKS];
    __shared__ sel_i32x4 codes[W][16 * D / 8];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int t = blockIdx.x / a.KVH, h = blockIdx.x - t * a.KVH, GQ = a.QH / a.KVH;
    const int32_t *tab = A.tables + (size_t)t * A.table_stride;
    const int nb = min(sel_blocks_of_row(A, t), BLOCKS);
    const int groups = (nb + 15) / 16;
    sel_i32x4 qa[KS];
    const int eq = sel_query<D>(A.q + ((size_t)t * a.QH + h * GQ + min(c & (A.P - 1), GQ - 1)) * D * 2, g, A.io_dtype, qa);
    float qm[4];
#pragma unroll
    for (int j = 0; j < 4; j++) qm[j] = sel_pow2(__shfl(eq, 4 * g + j));
    for (int g0 = w; g0 < groups; g0 += G * W) {
        int blk[G], e[G];
        sel_i32x4 bv[G][KS];
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int b = (g0 + i * W) * 16 + c;
            blk[i] = b < nb ? tab[b] : -1;
        }
#pragma unroll
        for (int i = 0; i < G; i++) {
            if (g0 + i * W >= groups) continue;                          // the same for the whole wave
            sel_fetch<D>(bv[i], A.bounds, a, h, blk[i], 0, lane);
            e[i] = (unsigned)blk[i] < (unsigned)a.NB ? (int)(int8_t)A.exps[(size_t)blk[i] * a.KVH + h] : kNoBlock;
        }
#pragma unroll
        for (int i = 0; i < G; i++) {
            if (g0 + i * W >= groups) continue;
            const int b = (g0 + i * W) * 16 + c;
            sel_wave_order();
            sel_stage<D>(codes[w], bv[i], lane);
            sel_wave_order();
            sel_i32x4 acc = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
            for (int k = 0; k < KS; k++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[k], sel_operand<D>(codes[w], k, g, c), acc, 0, 0, 0);
#endif
            const uint32_t x = sel_row_key(acc, qm, A.P, e[i] == kNoBlock ? 0.0f : sel_pow2(e[i]));
            if (g == 0) key_lds[b] = sel_key_of(A, x, b, nb, e[i]);
        }
    }
    __syncthreads();
    uint32_t kr[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int b = (w * NR + i) * 64 + lane;
        kr[i] = b < nb ? key_lds[b] : 0u;
    }
    topk_run<THREADS, NR, false>(S, kr, nb, A.keep, A.out + (size_t)blockIdx.x * A.keep, [](int, uint32_t (&)[NR]) {});
}

static unsigned sel_key_stride(const Lay &a, int max_seq_len)
{
    return (unsigned)(((size_t)max_seq_len + a.bs - 1) / a.bs + 3) & ~3u;
}

// Groups a workgroup of score_tile_kernel walks.  `rows` workgroups stand side by side; the context is cut into the number
// of parts that ends soonest: workgroups per CU, times a part's groups and its queries' conversion.  At head_dim 256 a CU holds
// one workgroup, below two and more, whose loads and products overlap by about a fifth; there a part is at most 64 groups
// (1 MiB of codes), so that the rows' workgroups stay near each other in the cache.  Against about 256 workgroups of at most 32 groups
// each: 1024 tokens x 4 heads x 256 at 16k 74 -> 51 us, 2048 tokens at 64k 343 -> 296 us.
static int sel_tile_groups(const Lay &a, unsigned groups, unsigned rows)
{
    const unsigned least = a.D <= 128 ? (groups + 63) / 64 : 1;
    unsigned best = 0xffffffffu, take = 4;
    for (unsigned parts = least; parts == least || (parts <= groups && rows * parts <= 4 * kSelTileWgs); parts++) {
        const unsigned g = ((groups + parts - 1) / parts + 3) & ~3u;
        const unsigned per_cu = (rows * ((groups + g - 1) / g) + kSelTileWgs - 1) / kSelTileWgs;
        const unsigned cost = (a.D <= 128 && per_cu > 1 ? 4 : 5) * per_cu * (g + kSelTileStart);
        if (cost < best) { best = cost; take = g; }
    }
    return (int)take;
}

template <int D>
static void launch_score(const Lay &a, const SelArgs &A, bool tile, dim3 grid, hipStream_t st)
{
    if constexpr (D <= 256) {
        if (tile) {
            if (A.P == 4) hipLaunchKernelGGL((score_tile_kernel<D, 2, 4>), grid, dim3(512), 0, st, a, A);
            else if (A.P == 8) hipLaunchKernelGGL((score_tile_kernel<D, 2, 8>), grid, dim3(512), 0, st, a, A);
            else hipLaunchKernelGGL((score_tile_kernel<D, 2, 16>), grid, dim3(512), 0, st, a, A);
            return;
        }
    }
    hipLaunchKernelGGL((score_kernel<D>), grid, dim3(256), 0, st, a, A);
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
    if (table_stride > 0 && (size_t)table_stride * a.bs < (size_t)max_seq_len) {        // no row is longer than its table
        max_seq_len = table_stride * a.bs;
        A.key_stride = sel_key_stride(a, max_seq_len);
    }
    A.bounds = (const uint8_t *)bounds + (size_t)layer * a.NB * a.KVH * 2 * a.D;
    A.exps = (const uint8_t *)bounds + bounds_exps_offset(a) + (size_t)layer * a.NB * a.KVH;
    A.q = (const uint8_t *)q; A.tables = d_tables; A.seq_lens = d_seq_lens; A.keys = (uint32_t *)workspace; A.out = d_selected;
    A.table_stride = table_stride; A.pos_start = pos_start; A.T = T; A.max_seq_len = max_seq_len;
    A.keep = n_keep; A.sink = n_sink; A.recent = n_recent; A.io_dtype = io_dtype;
    A.bs_div = mk_div((unsigned)a.bs);
    A.P = 4;
    while (A.P < a.QH / a.KVH) A.P *= 2;
    A.R = table_stride == 0 && T > 1 ? 16 / A.P : 1;
    // more than four sets of rows over one table; a workgroup stores the keys of its 64 rows at 32-bit byte offsets
    const bool tile = table_stride == 0 && a.D <= 256 && T > 4 * A.R && (size_t)a.KVH * A.key_stride <= (1u << 22);
    const int n = (int)(((size_t)max_seq_len + a.bs - 1) / a.bs);
    hipStream_t st = (hipStream_t)stream;
    if (n <= kSelShort || (n <= kSelFused && a.D <= 256 && !tile &&
                           ((size_t)n * 2 * a.D <= kSelFusedBytes || (size_t)T * a.KVH >= kSelFusedRows))) {
        const dim3 grid(T * a.KVH);
#define DRK_SELECT_LAUNCH(D)                                                                                                       \
    do {                                                                                                                           \
        if (n <= kSelShort) hipLaunchKernelGGL((select_kernel<D, 256, kSelShort>), grid, dim3(256), 0, st, a, A);                  \
        else hipLaunchKernelGGL((select_kernel<(D < 512 ? D : 256), 512, kSelFused>), grid, dim3(512), 0, st, a, A);               \
    } while (0)
        switch (a.D) {
        case 64: DRK_SELECT_LAUNCH(64); break;
        case 128: DRK_SELECT_LAUNCH(128); break;
        case 256: DRK_SELECT_LAUNCH(256); break;
        default: DRK_SELECT_LAUNCH(512); break;                      // short contexts only
        }
#undef DRK_SELECT_LAUNCH
        DRK_LAUNCH_CHECK("select_kernel");
        return DRK_OK;
    }
    if (n > 0) {
        const int rows = tile ? 16 * A.R : A.R;
        const size_t tiles = ((size_t)T + rows - 1) / rows, groups = ((size_t)n + 15) / 16;
        const size_t all = groups * a.KVH * tiles;                        // 16-block groups of every kv head and row tile
        if (tile) {
            A.groups_per_wave = sel_tile_groups(a, (unsigned)groups, (unsigned)(tiles * a.KVH));
        } else {
            const size_t units = a.D <= 128 ? kSelWaves : kSelWaves / 2;          // as many waves as should have work of their own
            const size_t gpw = (all + units - 1) / units;
            // (eight groups, with a second load of table entries: 16 branches x 64k 33.5 -> 35.7 us)
            A.groups_per_wave = (int)(gpw > kSelWaveGroups ? kSelWaveGroups : gpw);
        }
        const size_t per = (size_t)A.groups_per_wave * (tile ? 1 : 4);
        const size_t parts = (groups + per - 1) / per;
        if (tiles > 65535 || parts > 65535)
            return fail(DRK_ERR_UNSUPPORTED, "block_select: %d rows of %d blocks are more than one launch takes", T, n);
        const dim3 grid(a.KVH, (unsigned)parts, (unsigned)tiles);
        switch (a.D) {
        case 64: launch_score<64>(a, A, tile, grid, st); break;
        case 128: launch_score<128>(a, A, tile, grid, st); break;
        case 256: launch_score<256>(a, A, tile, grid, st); break;
        default: launch_score<512>(a, A, tile, grid, st); break;
        }
        DRK_LAUNCH_CHECK("score_kernel");
    }
    const dim3 rows(T * a.KVH);
    // Keys in one slab of registers.  Few rows: twice the threads, half the keys each (8 rows of 2048 keys, with the scores, 10.4 -> 9.0 us);
    // many rows keep the chip busy by themselves, so fewer threads, whose steps are less exchange: 8192 rows of 4100 keys with their
    // scores 162 us with 1024 threads, 114 with 512, 103 with 256; but below 2048 keys 128 threads cost 2048 rows 1 us more than 256.
    const bool few = T * a.KVH <= 512;
#define DRK_TOPK_LAUNCH(THREADS, NR, MULTI) hipLaunchKernelGGL((topk_kernel<THREADS, NR, MULTI>), rows, dim3(THREADS), 0, st, A, a.KVH)
    if (n > 8192) DRK_TOPK_LAUNCH(1024, 8, true);
    else if (n > 4096 && few) DRK_TOPK_LAUNCH(1024, 8, false);
    else if (n > 4096) DRK_TOPK_LAUNCH(512, 16, false);
    else if (n > 2048 && few) DRK_TOPK_LAUNCH(1024, 4, false);
    else if (n > 2048) DRK_TOPK_LAUNCH(256, 16, false);
    else if (few) DRK_TOPK_LAUNCH(512, 4, false);
    else DRK_TOPK_LAUNCH(256, 8, false);
#undef DRK_TOPK_LAUNCH
    DRK_LAUNCH_CHECK("topk_kernel");
    return DRK_OK;
}

} // extern "C"
