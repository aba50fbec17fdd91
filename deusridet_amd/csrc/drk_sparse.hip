// drk_sparse.hip -- paged GQA attention over the blocks a selection lists for each (row, kv head).
//
// The listed blocks' tokens are one long axis, cut into groups of 16 (a block is a whole number of
// them).  A workgroup of eight waves takes a piece of one (row, kv head)'s groups -- or, where rows abound, two,
// four or eight whole rows: first every thread turns a few groups into descriptors in LDS -- list entry, block
// table, page offset: the dependent loads happen there, side by side, and groups without a token drop
// out -- then the waves walk them independently, each with a running maximum and sum per query head and the
// output in registers:
//   S[token][head] = K[16 x D] Q^T       D/32 x v_mfma_f32_16x16x32
//   O[head][dim]  += P[heads x 16] V     D/16 x v_mfma_f32_16x16x16
// with the query heads of the group as the 16-wide operand.  The waves' states meet at the end; a row
// that was cut leaves (o, m, l) per piece for sparse_merge_kernel, otherwise it is written at once.
//
// Bound by HBM for branches: 64 x 256 blocks of 16 tokens x 8 heads x 128 (1.08 GB bf16) 169 us, 6.4 TB/s (183 with other pages
// every time: translations); 16 x 128 blocks int8 (69 MB) 17 us, of which the walk is 10, the rest launch, list, table,
// first pages and the end, + 4 for the merge; 1 x 64 blocks 6 + 3 us, all of it latency.  Rows of a chunk meet in the L2
// instead: 512 x 64 blocks (2.1 GB from 134 MB of pages) 126 us, 17 TB/s, two thirds of the lines from the L2; lists that
// all stay in it 83 us, 26 TB/s.
#include "drk_stream_tile.hpp"

namespace drk {

constexpr int kSpGroups = 512;          // 16-token groups one workgroup may own (descriptors in LDS)
constexpr int kSpMaxPieces = 64;        // pieces of a row: a lane each in the merge
constexpr int kSpWaves = 8;             // waves of a workgroup
constexpr size_t kSpUncut = 32 * 128;   // groups times head_dim up to which a row is not cut
constexpr int kSpWgs = 512;             // workgroups of head_dim 128 a launch aims at: the 2 a CU holds (head_dim 256: half)

struct SparseArgs {
    const uint8_t *pool_layer, *q;
    const int32_t *tables, *seq_lens, *sel;
    const uint16_t *gate;
    uint16_t *out;
    float *part_o, *part_m, *part_l;     // [T][QH][pieces]([D])
    size_t gate_stride;
    int table_stride, table_blocks, pos_start, T, KVH, QH, NB, bs, keep, io_dtype;
    int pieces, groups_per_piece, groups;    // 16-token groups of a (row, kv head)'s list
    unsigned head_stride, kv_plane, block_stride, scale_plane, row_bytes;
    float scale_log2e;
};

// The second product takes its weights in the 16-bit type its values come in (8-bit pages: fp16), rounded to nearest: a
// 32-bit product would cost eight times the matrix instructions.  bf16 has fp32's range.  fp16 ends at 2^-24, and a wave may walk
// 8192 tokens whose small weights count together: the largest weight is taken as 2^14 instead of 1, so that only what
// is 2^39 below it vanishes.  With int8 pages the weight is p times the token's V scale, and all V scales may be 2^-14
// or less: there the reference follows the largest p * scale, so that the product's weights fill the same range
// whatever the scales are (p itself and its sum are in 32 bits).  Following p alone, a token 8 nats ahead of 2048 others with
// scales of 2^-16 took their share of the output to nought; the time is the same (16 x 128 blocks int8 21.1 us).
template <int DOT> constexpr float kSpHeadroom = DOT == DRK_BF16 ? 0.0f : 14.0f;

// log2 of a V scale's magnitude, kept finite: nought (whose token only counts in the sum), infinity and NaN must not
// become the reference
__device__ __forceinline__ float sparse_log2_scale(float vs)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return fminf(fmaxf(__builtin_amdgcn_logf(fabsf(vs)), -24.0f), 16.0f);
#else
    return vs;
#endif
}

// what a workgroup keeps in LDS beside the staged keys: the rows' query heads and group descriptors
struct SparseLds {
    unsigned q, desc, total;             // bytes per row of queries / of descriptors (offsets, scale offsets, counts), all
    unsigned soff, cnt;                  // where they begin inside a row's descriptors
};
__host__ __device__ inline SparseLds sparse_lds(int GQ, int pitch, int groups, bool scales, int rows)
{
    SparseLds s;
    s.q = (unsigned)(GQ * pitch);
    s.soff = (unsigned)groups * 4;
    s.cnt = s.soff * (scales ? 2 : 1);
    s.desc = (s.cnt + (unsigned)groups + 15) & ~15u;
    s.total = (s.q + s.desc) * (unsigned)rows;
    return s;
}

// WPR waves per row.  More than one: a row's waves take every WPR-th group and fold their states at the end.
template <int DT, int D, bool NT, int WPR>
__global__ __launch_bounds__(kSpWaves * 64, D == 128 ? 4 : 2) void sparse_kernel(SparseArgs A)
{
    using Geo = StreamGeo<DT, D>;
    [[maybe_unused]] constexpr bool Q8 = Geo::q8;
    constexpr int DOT = KvTraits<DT>::dot;
    constexpr int W = WPR, ROWS = kSpWaves / WPR, RT = WPR * 64;      // RT: threads per row
    __shared__ __align__(16) uint8_t k_lds[kSpWaves][16 * Geo::PITCH];   // the waves' staged keys; at the end their outputs
    __shared__ float mw_all[kSpWaves][16], lw_all[kSpWaves][16];
    __shared__ int wcount[kSpWaves];
    extern __shared__ __align__(16) uint8_t dyn_lds[];
    static_assert(sizeof(k_lds) >= kSpWaves * 4 * D * sizeof(float), "the waves' outputs of one round fit over the keys");

    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int rw = wave / WPR, w = wave - rw * WPR;                   // row of the workgroup, wave of the row
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15, rtid = w * 64 + lane;
    const int GQ = A.QH / A.KVH;
    // kv heads vary fastest: neighbouring workgroups, on different XCDs, read different heads' rows
    const int h = (int)(blockIdx.x % (unsigned)A.KVH), tp = (int)(blockIdx.x / (unsigned)A.KVH);
    const int t = (tp / A.pieces) * ROWS + rw, piece = tp - (tp / A.pieces) * A.pieces;
    const bool row_on = t < A.T;
    const int len = row_on ? (A.seq_lens ? A.seq_lens[t] : A.pos_start + t + 1) : 0;
    const int bq = t * A.QH + h * GQ;
    const SparseLds S = sparse_lds(GQ, Geo::PITCH, A.groups_per_piece, DT == DRK_INT8, ROWS);
    uint8_t *const q_lds = dyn_lds + rw * S.q, *const desc = dyn_lds + ROWS * S.q + rw * S.desc;
    uint32_t *const goff = (uint32_t *)desc, *const gsoff = (uint32_t *)(desc + S.soff);
    uint8_t *const gcnt = desc + S.cnt;
    float (*const mw_lds)[16] = mw_all + rw * WPR, (*const lw_lds)[16] = lw_all + rw * WPR;
    float (*const o_lds)[4][D] = (float (*)[4][D]) & k_lds[0][0] + rw * WPR;

    // ---- the query heads, on their way while the descriptors are built ----
    constexpr int QL = (16 * (D / 8) + RT - 1) / RT;                  // at most 16 heads of 16-byte chunks
    uint4 qv[QL];
    const int qn = row_on ? GQ * (D / 8) : 0;
    const uint8_t *const qsrc = A.q + (size_t)(row_on ? bq : 0) * (D * 2);
#pragma unroll
    for (int i = 0; i < QL; i++)
        if (rtid + i * RT < qn) qv[i] = *(const uint4 *)(qsrc + (size_t)(rtid + i * RT) * 16);

    // ---- descriptors of the groups that hold tokens, in order ----
    const int32_t *sel = A.sel + ((size_t)t * A.KVH + h) * A.keep;
    const int32_t *tab = A.tables + (size_t)t * A.table_stride;
    const int g0 = piece * A.groups_per_piece, gn = min(A.groups_per_piece, A.groups - g0), gpb = A.bs / 16;
    int n = 0;
    for (int i0 = 0; i0 < gn; i0 += RT) {
        const int gi = g0 + i0 + rtid;
        uint32_t off = 0, soff = 0;
        int cnt = 0;
        if (i0 + rtid < gn && len > 0) {
            const int e = gi / gpb, lb = sel[e], p0 = (gi - e * gpb) * 16;
            if (lb >= 0 && lb <= (len - 1) / A.bs && lb < A.table_blocks) {
                cnt = min(16, len - lb * A.bs - p0);
                if (cnt > 0) {
                    const int blk = tab[lb];
                    if (blk >= 0 && blk < A.NB) {
                        const size_t base = (size_t)blk * A.block_stride;
                        off = (uint32_t)((base + (size_t)h * A.head_stride + (size_t)p0 * A.row_bytes) >> 4);
                        soff = (uint32_t)((base + 2 * (size_t)A.kv_plane + ((size_t)h * A.bs + p0) * 2) >> 4);
                    } else {
                        cnt = 0;
                    }
                }
            }
        }
        const uint64_t live = __ballot(cnt > 0);
        int at = n + __popcll(live & ((1ull << lane) - 1));
        if constexpr (WPR > 1) {
            if (lane == 0) wcount[wave] = __popcll(live);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < W; i++) {
                if (i < w) at += wcount[rw * WPR + i];
                n += wcount[rw * WPR + i];
            }
        } else {
            n += __popcll(live);
        }
        if (cnt > 0) {
            goff[at] = off;
            gcnt[at] = (uint8_t)cnt;
            if (DT == DRK_INT8) gsoff[at] = soff;
        }
        if (WPR > 1) __syncthreads();                                 // the counts have been read
    }

#pragma unroll
    for (int i = 0; i < QL; i++) {
        const int x = rtid + i * RT, r = x / (D / 8), ch = x - r * (D / 8);
        if (x >= qn) continue;
        uint4 v = qv[i];
#if defined(__HIP_DEVICE_COMPILE__)
        if (Q8 && A.io_dtype == DRK_BF16) {                           // quantised pages multiply in fp16
            v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_lo(v.x), bf16_hi(v.x)));
            v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_lo(v.y), bf16_hi(v.y)));
            v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_lo(v.z), bf16_hi(v.z)));
            v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_lo(v.w), bf16_hi(v.w)));
        }
#endif
        *(uint4 *)(q_lds + r * Geo::PITCH + ch * 16) = v;
    }
    __syncthreads();
    // operand rows GQ .. 15 repeat the last head: what comes out of them is not used
    const uint8_t *const qrow = q_lds + min(c, GQ - 1) * Geo::PITCH + g * 16;
    float qbias = 0.0f;
    if (DT == DRK_INT8) {                                             // sum of the head's query values, for the code offset
        float sq = 0.0f;
#pragma unroll
        for (int kk = 0; kk < Geo::NQK; kk++) {
            const uint4 v = *(const uint4 *)(qrow + kk * 64);
            sq = s_dot2<DOT>(v.x, kF16Ones, sq);
            sq = s_dot2<DOT>(v.y, kF16Ones, sq);
            sq = s_dot2<DOT>(v.z, kF16Ones, sq);
            sq = s_dot2<DOT>(v.w, kF16Ones, sq);
        }
        sq += __shfl_xor(sq, 16);
        sq += __shfl_xor(sq, 32);
        qbias = kI8Bias * sq;
    }

    w_f32x4 o[Geo::NPV];
#pragma unroll
    for (int e = 0; e < Geo::NPV; e++) o[e] = w_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_lane = 0.0f, ps_lane = 0.0f;
    uint8_t *const klds = &k_lds[wave][0];
    auto load_scales = [&](int i, uint2 &ks, uint2 &vs) {
        if (DT != DRK_INT8) return;
        const uint8_t *p = A.pool_layer + ((size_t)gsoff[i] << 4) + g * 8;
        ks = *(const uint2 *)p;
        vs = *(const uint2 *)(p + A.scale_plane);
    };

    KRegs<DT, D> kreg = {};
    VRegs<DT, D> vreg = {};
    uint2 ksr = {}, vsr = {};
    if (w < n) {
        kreg = load_k<DT, D, NT>(A.pool_layer, goff[w], lane);
        vreg = load_v<DT, D, NT>(A.pool_layer, goff[w], A.kv_plane, lane);
        load_scales(w, ksr, vsr);
    }
    for (int i = w; i < n; i += W) {
        const int lim = __builtin_amdgcn_readfirstlane((int)gcnt[i]);
        const bool more = i + W < n;
        stage_k<DT, D>(klds, kreg, lane);
        [[maybe_unused]] const uint2 ksc = ksr, vsc = vsr;     // packed until the softmax: registers
        uint32_t next = 0;
        if (more) {
            next = goff[i + W];
            kreg = load_k<DT, D, NT>(A.pool_layer, next, lane);
            load_scales(i + W, ksr, vsr);
        }
        w_f32x4 sacc = {0.0f, 0.0f, 0.0f, 0.0f};
        const uint8_t *arow = klds + c * Geo::PITCH + g * 16;
#pragma unroll
        for (int k0 = 0; k0 < Geo::NQK; k0 += 4) {
            uint4 ka[4], qa[4];
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
                ka[kk] = *(const uint4 *)(arow + (k0 + kk) * 64);
                qa[kk] = *(const uint4 *)(qrow + (k0 + kk) * 64);
            }
#pragma unroll
            for (int kk = 0; kk < 4; kk++) sacc = w_mfma_qk<DOT>(ka[kk], qa[kk], sacc);
        }
        // softmax of head c over tokens 4g..4g+3 (+ the other three lane groups): weights are 2^(sc - m_ref), m_ref the largest
        // `top` so far less kSpHeadroom
        const int t0 = g * 4;
        float sc[4], top[4], p[4], vs[4] = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x = sacc[j];
            if (DT == DRK_INT8) {
                x = (x - qbias) * f16_bits_to_f((uint16_t)((j < 2 ? ksc.x : ksc.y) >> (16 * (j & 1)) & 0xffffu));
                vs[j] = f16_bits_to_f((uint16_t)((j < 2 ? vsc.x : vsc.y) >> (16 * (j & 1)) & 0xffffu));
            }
            x *= A.scale_log2e;
            sc[j] = t0 + j < lim ? x : -INFINITY;
            top[j] = DT == DRK_INT8 ? sc[j] + sparse_log2_scale(vs[j]) : sc[j];
        }
        float mloc = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        mloc = fmaxf(mloc, __shfl_xor(mloc, 16));
        mloc = fmaxf(mloc, __shfl_xor(mloc, 32));
        const float m_new = fmaxf(m_run, mloc), m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = s_exp2(m_run - m_use), m_ref = m_use - kSpHeadroom<DOT>;
        m_run = m_new;
        float pw[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p[j] = s_exp2(sc[j] - m_ref);
            pw[j] = DT == DRK_INT8 ? (t0 + j < lim ? p[j] * vs[j] : 0.0f) : p[j];
        }
        uint2 pa;                                             // P[head c][tokens 4g..4g+3] for the second product
        if constexpr (DOT == DRK_BF16) {
            pa.x = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)pw[0]) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)pw[1]) << 16);
            pa.y = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)pw[2]) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)pw[3]) << 16);
        } else {
            pa.x = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)pw[0]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)pw[1]) << 16);
            pa.y = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)pw[2]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)pw[3]) << 16);
        }
        // the denominator sums the rounded weights the product multiplies, so both carry the same rounding
        // (int8: the product multiplies p times the V scale; its own sum takes the code offset out again)
        float rs;
        if (DT == DRK_INT8) {
            float tsum = s_dot2<DOT>(pa.x, kF16Ones, 0.0f);
            tsum = s_dot2<DOT>(pa.y, kF16Ones, tsum);
            ps_lane = fmaf(ps_lane, alpha, tsum);
            rs = (p[0] + p[1]) + (p[2] + p[3]);
        } else {
            const uint32_t ones = DOT == DRK_BF16 ? kBf16Ones : kF16Ones;
            rs = s_dot2<DOT>(pa.y, ones, s_dot2<DOT>(pa.x, ones, 0.0f));
        }
        l_lane = fmaf(l_lane, alpha, rs);
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
            const float a0 = __shfl(alpha, 4 * g), a1 = __shfl(alpha, 4 * g + 1);
            const float a2 = __shfl(alpha, 4 * g + 2), a3 = __shfl(alpha, 4 * g + 3);
#pragma unroll
            for (int e = 0; e < Geo::NPV; e++) { o[e][0] *= a0; o[e][1] *= a1; o[e][2] *= a2; o[e][3] *= a3; }
        }
        if (DT != DRK_INT8 && lim < 16) {                     // rows without a token may hold anything (NaN)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (t0 + j >= lim) {
#pragma unroll
                    for (int ch = 0; ch < Geo::NCH; ch++) vreg.r[j][ch] = {};
                }
        }
#pragma unroll
        for (int ch = 0; ch < Geo::NCH; ch++) {
            uint2 vb[8];
            v_operands<DT>(vreg.r[0][ch], vreg.r[1][ch], vreg.r[2][ch], vreg.r[3][ch], vb);
#pragma unroll
            for (int e = 0; e < 8; e++) o[ch * 8 + e] = w_mfma_pv<DOT>(pa, vb[e], o[ch * 8 + e]);
        }
        if (more) vreg = load_v<DT, D, NT>(A.pool_layer, next, A.kv_plane, lane);
    }

    // ---- the end: fold the waves ----
    float lw = l_lane, psum = ps_lane;
    lw += __shfl_xor(lw, 16);
    lw += __shfl_xor(lw, 32);
    if (DT == DRK_INT8) {
        psum += __shfl_xor(psum, 16);
        psum += __shfl_xor(psum, 32);
    }
    if constexpr (WPR == 1) {
        // nothing to fold: head 4g + j, dims ch * 128 + 8c .. + 7 are in this lane
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int hh = 4 * g + j;
            const float L = __shfl(lw, hh), bias = DT == DRK_INT8 ? kI8Bias * __shfl(psum, hh) : 0.0f;
            if (hh >= GQ || !row_on || L == 0.0f) continue;
#pragma unroll
            for (int ch = 0; ch < Geo::NCH; ch++) {
                const int d = ch * 128 + c * 8;
                const uint16_t *gp = A.gate ? A.gate + (size_t)(bq + hh) * A.gate_stride + d : nullptr;
                uint4 gv = make_uint4(0u, 0u, 0u, 0u);
                if (gp) gv = *(const uint4 *)gp;
                const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float v = (o[ch * 8 + e][j] - bias) / L;
                    if (gp) v = sigmoid_gate_value(v, elem16_to_f((uint16_t)(gw[e >> 1] >> (16 * (e & 1))), A.io_dtype));
                    const uint32_t b16 = f_to_elem16(v, A.io_dtype);
                    y[e >> 1] = e & 1 ? y[e >> 1] | b16 << 16 : b16;
                }
                *(uint4 *)(A.out + (size_t)(bq + hh) * D + d) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
        return;
    }
    if (lane < 16) { mw_lds[w][lane] = m_run; lw_lds[w][lane] = lw; }
    __syncthreads();                                          // (the staged keys have been read, too)
    float f_own[4], bias[4];                                  // this wave's weight / code offset for head 4g + j
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int hh = 4 * g + j;
        float M = mw_lds[0][hh];
#pragma unroll
        for (int i = 1; i < W; i++) M = fmaxf(M, mw_lds[i][hh]);
        const float mo = mw_lds[w][hh];
        f_own[j] = mo == -INFINITY ? 0.0f : s_exp2(mo - M);
        bias[j] = DT == DRK_INT8 ? kI8Bias * __shfl(psum, hh) : 0.0f;
    }
    // 4 heads per round, whose dims the row's threads share out
    constexpr int VEC = D / 128, UNITS = 4 * (D / VEC) / RT;  // dims per thread at a time, times per round
    for (int r = 0; r < (GQ + 3) >> 2; r++) {
        if (r > 0) __syncthreads();
        if (g == r) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int ch = 0; ch < Geo::NCH; ch++) {
                    float *dst = &o_lds[w][j][ch * 128 + c * 8];
                    const w_f32x4 *oc = &o[ch * 8];
                    *(float4 *)dst = make_float4((oc[0][j] - bias[j]) * f_own[j], (oc[1][j] - bias[j]) * f_own[j],
                                                 (oc[2][j] - bias[j]) * f_own[j], (oc[3][j] - bias[j]) * f_own[j]);
                    *(float4 *)(dst + 4) = make_float4((oc[4][j] - bias[j]) * f_own[j], (oc[5][j] - bias[j]) * f_own[j],
                                                       (oc[6][j] - bias[j]) * f_own[j], (oc[7][j] - bias[j]) * f_own[j]);
                }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int x = rtid + u * RT, hr = x / (D / VEC), hh = 4 * r + hr, d = (x - hr * (D / VEC)) * VEC;
            if (hh >= GQ || !row_on) continue;
            float M = mw_lds[0][hh], L = 0.0f;
#pragma unroll
            for (int i = 1; i < W; i++) M = fmaxf(M, mw_lds[i][hh]);
#pragma unroll
            for (int i = 0; i < W; i++) {
                const float ll = lw_lds[i][hh];
                if (ll != 0.0f) L = fmaf(ll, s_exp2(mw_lds[i][hh] - M), L);   // (a NaN takes part)
            }
            float acc[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                acc[e] = 0.0f;
#pragma unroll
                for (int i = 0; i < W; i++) acc[e] += o_lds[i][hr][d + e];
            }
            if (A.pieces > 1) {
                const size_t pi = (size_t)(bq + hh) * A.pieces + piece;
#pragma unroll
                for (int e = 0; e < VEC; e++) A.part_o[pi * D + d + e] = acc[e];
                if (d == 0) { A.part_m[pi] = M; A.part_l[pi] = L; }
            } else if (L != 0.0f) {
                uint16_t *dst = A.out + (size_t)(bq + hh) * D + d;
                const uint16_t *gp = A.gate ? A.gate + (size_t)(bq + hh) * A.gate_stride + d : nullptr;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    float y = acc[e] / L;
                    if (gp) y = sigmoid_gate_value(y, elem16_to_f(gp[e], A.io_dtype));
                    dst[e] = f_to_elem16(y, A.io_dtype);
                }
            }
        }
    }
}

// grid T * QH, one wave: lane s owns the weight of piece s
template <int D>
__global__ __launch_bounds__(64) void sparse_merge_kernel(SparseArgs A)
{
    constexpr int VEC = D / 64;
    const size_t row = blockIdx.x, base = row * A.pieces;
    const int lane = threadIdx.x, d = lane * VEC;
    const bool mine = lane < A.pieces;
    const float m = mine ? A.part_m[base + lane] : -INFINITY, l = mine ? A.part_l[base + lane] : 0.0f;
    const bool live = l != 0.0f;                               // (a NaN takes part)
    const float M = s_wave_max(live ? m : -INFINITY);
    if (__ballot(live) == 0) return;                           // no token took part
    const float wgt = live ? s_exp2(m - M) : 0.0f;
    const float L = s_wave_sum(live ? l * wgt : 0.0f);
    typedef float fvec __attribute__((ext_vector_type(VEC)));
    fvec acc = {};
    for (int s0 = 0; s0 < A.pieces; s0 += 8) {                 // eight rows in flight
        fvec o[8];
        float ws[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int s = min(s0 + u, A.pieces - 1);
            ws[u] = s0 + u < A.pieces ? s_lane(wgt, s) : 0.0f;
            o[u] = *(const fvec *)(A.part_o + (base + s) * D + d);
        }
#pragma unroll
        for (int u = 0; u < 8; u++)
#pragma unroll
            for (int x = 0; x < VEC; x++) acc[x] = fmaf(o[u][x], ws[u], acc[x]);
    }
    uint16_t *dst = A.out + row * D + d;
    const uint16_t *gp = A.gate ? A.gate + row * A.gate_stride + d : nullptr;
#pragma unroll
    for (int x = 0; x < VEC; x++) {
        float y = acc[x] / L;
        if (gp) y = sigmoid_gate_value(y, elem16_to_f(gp[x], A.io_dtype));
        dst[x] = f_to_elem16(y, A.io_dtype);
    }
}

// Pieces of a (row, kv head): enough workgroups for the chip, but no piece shorter than a group per wave and none
// longer than the descriptor table.  A cut costs a second launch and the merge, about 3 us, so a short list is walked
// by one workgroup: one row of 8 kv heads x 128, 32 groups each, 9.3 us instead of 10.5 -- but 64 groups 16 instead
// of 10 (with 16 waves in the workgroup), and at head_dim 256, whose groups are twice the bytes, 32 groups 15.5
// instead of 11.6.
static int sparse_pieces(const Lay &a, int T, int n_keep, int *groups_per_piece)
{
    const size_t groups = (size_t)n_keep * (a.bs / 16), rows = (size_t)T * a.KVH;
    size_t p = (kSpWgs * 128 / a.D + rows - 1) / rows;
    p = p > (groups + kSpWaves - 1) / kSpWaves ? (groups + kSpWaves - 1) / kSpWaves : p;
    p = p > kSpMaxPieces ? kSpMaxPieces : p;
    if (groups * a.D <= kSpUncut) p = 1;
    const size_t least = (groups + kSpGroups - 1) / kSpGroups;
    p = p < least ? least : p;
    if (p > kSpMaxPieces) return 0;
    *groups_per_piece = (int)((groups + p - 1) / p);
    return (int)((groups + *groups_per_piece - 1) / *groups_per_piece);
}

// Waves per row: as few as still give the chip the waves it holds (16 per CU at head_dim 128, 8 at 256) and leave
// room in LDS for that many: fewer waves per row, fewer states to fold (512 rows x 64 blocks: one wave 128 us, eight 183).
static int sparse_waves_per_row(const Lay &a, int T, int groups_per_piece)
{
    const size_t rows = (size_t)T * a.KVH, waves = a.D == 128 ? 4096 : 2048;
    const unsigned pitch = (unsigned)a.D * 2 + 16, staged = kSpWaves * 16 * pitch + 2048, room = (a.D == 128 ? 80u : 160u) << 10;
    int w = 8;
    while (w > 1 && rows * (w / 2) >= waves &&
           staged + sparse_lds(a.QH / a.KVH, (int)pitch, groups_per_piece, a.dtype == DRK_INT8, kSpWaves / (w / 2)).total <= room)
        w /= 2;
    return w;
}

static int sparse_check(const drk_kv_layout *g, Lay *a, int T, int n_keep, int *pieces, int *gpp, const char *who)
{
    int rc = make_lay(g, a);
    if (rc) return rc;
    if ((a->D != 128 && a->D != 256) || (a->bs % 16) || a->QH / a->KVH > 16)
        return fail(DRK_ERR_UNSUPPORTED, "%s: head_dim 128 or 256, block_size a multiple of 16 and at most 16 query heads per kv "
                    "head are supported (head_dim %d, block_size %d, %d heads)", who, a->D, a->bs, a->QH / a->KVH);
    if ((a->layer_stride >> 4) > 0xfffffffeu) return fail(DRK_ERR_UNSUPPORTED, "%s: one layer of the pool exceeds 64 GiB", who);
    if (T < 0 || n_keep < 1) return fail(DRK_ERR_INVALID, "%s: T %d, n_keep %d", who, T, n_keep);
    *pieces = *gpp = 1;
    if (T == 0) return DRK_OK;
    *pieces = sparse_pieces(*a, T, n_keep, gpp);
    if (*pieces == 0) return fail(DRK_ERR_UNSUPPORTED, "%s: n_keep %d blocks of %d tokens: at most %d tokens per row", who, n_keep, a->bs,
                                  kSpMaxPieces * kSpGroups * 16);
    if ((size_t)T * *pieces * a->KVH > 0x7fffffffu || (size_t)T * a->QH > 0x7fffffffu)
        return fail(DRK_ERR_UNSUPPORTED, "%s: T %d is more than one launch takes", who, T);
    return DRK_OK;
}

static int sparse_check_io(const Lay &a, int io_dtype, const char *who)
{
    if (io_dtype != DRK_F16 && io_dtype != DRK_BF16) return fail(DRK_ERR_INVALID, "%s: io_dtype must be F16 or BF16", who);
    if (a.E == 2 && io_dtype != a.dtype) return fail(DRK_ERR_INVALID, "%s: io_dtype %d differs from the pool's %d", who, io_dtype, a.dtype);
    return DRK_OK;
}

static size_t sparse_need(const Lay &a, int T, int pieces)
{
    return pieces > 1 ? (size_t)T * a.QH * pieces * (a.D + 2) * 4 : 0;
}

} // namespace drk

using namespace drk;

extern "C" {

size_t drk_paged_sparse_workspace_bytes(const drk_kv_layout *g, int T, int n_keep)
{
    Lay a;
    int pieces, gpp;
    if (sparse_check(g, &a, T, n_keep, &pieces, &gpp, "paged_sparse_workspace_bytes")) return 0;
    return sparse_need(a, T, pieces);
}

int drk_paged_sparse_check(const drk_kv_layout *g, int T, int n_keep, int io_dtype)
{
    Lay a;
    int pieces, gpp;
    const int rc = sparse_check(g, &a, T, n_keep, &pieces, &gpp, "paged_sparse_check");
    return rc ? rc : sparse_check_io(a, io_dtype, "paged_sparse_check");
}

int drk_paged_sparse_attention(const drk_kv_layout *g, const void *q, const void *pool, const int32_t *d_tables, int table_stride,
                               const int32_t *d_seq_lens, int pos_start, int T, const int32_t *d_selected, int n_keep, void *out,
                               int layer, float scale, int io_dtype, const void *gate, size_t gate_stride, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    Lay a;
    SparseArgs A;
    int rc = sparse_check(g, &a, T, n_keep, &A.pieces, &A.groups_per_piece, "paged_sparse_attention");
    if (rc) return rc;
    rc = sparse_check_io(a, io_dtype, "paged_sparse_attention");
    if (rc) return rc;
    if (layer < 0 || layer >= a.L) return fail(DRK_ERR_INVALID, "paged_sparse_attention: layer %d outside [0,%d)", layer, a.L);
    if (table_stride < 0 || pos_start < 0 || pos_start > 0x7fffffff - T || !(scale > 0.0f))
        return fail(DRK_ERR_INVALID, "paged_sparse_attention: bad argument");
    if (T == 0) return DRK_OK;
    if (!q || !pool || !d_tables || !d_selected || !out) return fail(DRK_ERR_INVALID, "paged_sparse_attention: NULL pointer");
    if (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out | (uintptr_t)workspace | (uintptr_t)gate) & 15u)
        return fail(DRK_ERR_INVALID, "paged_sparse_attention: q, pool, out, gate and the workspace must be 16-byte aligned");
    if (gate && (gate_stride < (size_t)a.D || (gate_stride % 8)))
        return fail(DRK_ERR_INVALID, "paged_sparse_attention: gate_stride %zu must be a multiple of 8, at least head_dim", gate_stride);
    const size_t need = sparse_need(a, T, A.pieces);
    if (need && (!workspace || workspace_bytes < need))
        return fail(DRK_ERR_WORKSPACE, "paged_sparse_attention: %zu bytes of workspace, %zu needed", workspace_bytes, need);
    A.pool_layer = (const uint8_t *)pool + (size_t)layer * a.layer_stride;
    A.q = (const uint8_t *)q; A.tables = d_tables; A.seq_lens = d_seq_lens; A.sel = d_selected;
    A.gate = (const uint16_t *)gate; A.gate_stride = gate_stride; A.out = (uint16_t *)out;
    const size_t np = (size_t)T * a.QH * A.pieces;
    A.part_o = (float *)workspace; A.part_m = A.part_o + np * a.D; A.part_l = A.part_m + np;
    A.table_stride = table_stride; A.table_blocks = table_stride > 0 ? table_stride : 0x7fffffff; A.pos_start = pos_start; A.T = T; A.KVH = a.KVH; A.QH = a.QH; A.NB = a.NB; A.bs = a.bs;
    A.keep = n_keep; A.io_dtype = io_dtype; A.groups = n_keep * (a.bs / 16);
    A.head_stride = a.head_stride; A.kv_plane = a.kv_plane; A.block_stride = a.block_stride; A.scale_plane = a.scale_plane;
    A.row_bytes = a.row_bytes;
    A.scale_log2e = scale * kSLog2e;
    hipStream_t st = (hipStream_t)stream;
    // rows over one table meet in the same pages: keep them cached (512 rows 128 us, non-temporal 244); branches do not
    // (64 x 256 blocks non-temporal 191, cached 210)
    const bool shared = table_stride == 0 && T > 1;
    const int wpr = A.pieces > 1 ? 8 : sparse_waves_per_row(a, T, A.groups_per_piece);
    const int per_wg = kSpWaves / wpr;                        // rows of a workgroup
    const dim3 grid((unsigned)(((size_t)T + per_wg - 1) / per_wg * A.pieces * a.KVH));
#define DRK_SPARSE_LAUNCH4(DT, D, NT, WPR)                                                                                  \
    hipLaunchKernelGGL((sparse_kernel<DT, D, NT, WPR>), grid, dim3(kSpWaves * 64),                              \
                       sparse_lds(a.QH / a.KVH, StreamGeo<DT, D>::PITCH, A.groups_per_piece, DT == DRK_INT8, per_wg).total, st, A)
#define DRK_SPARSE_LAUNCH3(DT, D, NT)                                                                                       \
    do {                                                                                                                    \
        if (wpr == 8) DRK_SPARSE_LAUNCH4(DT, D, NT, 8);                                                                \
        else if (wpr == 4) DRK_SPARSE_LAUNCH4(DT, D, NT, 4);                                                                \
        else if (wpr == 2) DRK_SPARSE_LAUNCH4(DT, D, NT, 2);                                                                \
        else DRK_SPARSE_LAUNCH4(DT, D, NT, 1);                                                                              \
    } while (0)
#define DRK_SPARSE_LAUNCH2(DT, D)                                                                                           \
    do {                                                                                                                    \
        if (shared) DRK_SPARSE_LAUNCH3(DT, D, false);                                                                       \
        else DRK_SPARSE_LAUNCH3(DT, D, true);                                                                               \
    } while (0)
#define DRK_SPARSE_LAUNCH(DT)                                                                                               \
    do {                                                                                                                    \
        if (a.D == 128) DRK_SPARSE_LAUNCH2(DT, 128);                                                                        \
        else DRK_SPARSE_LAUNCH2(DT, 256);                                                                                   \
    } while (0)
    switch (a.dtype) {
    case DRK_F16: DRK_SPARSE_LAUNCH(DRK_F16); break;
    case DRK_BF16: DRK_SPARSE_LAUNCH(DRK_BF16); break;
    case DRK_INT8: DRK_SPARSE_LAUNCH(DRK_INT8); break;
    default: DRK_SPARSE_LAUNCH(DRK_FP8_E4M3); break;
    }
#undef DRK_SPARSE_LAUNCH
#undef DRK_SPARSE_LAUNCH2
#undef DRK_SPARSE_LAUNCH3
#undef DRK_SPARSE_LAUNCH4
    DRK_LAUNCH_CHECK("sparse_kernel");
    if (A.pieces > 1) {
        if (a.D == 128) hipLaunchKernelGGL((sparse_merge_kernel<128>), dim3(T * a.QH), dim3(64), 0, st, A);
        else hipLaunchKernelGGL((sparse_merge_kernel<256>), dim3(T * a.QH), dim3(64), 0, st, A);
        DRK_LAUNCH_CHECK("sparse_merge_kernel");
    }
    return DRK_OK;
}

} // extern "C"
