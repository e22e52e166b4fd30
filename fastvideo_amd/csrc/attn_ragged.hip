// Ragged attention for BLOCKS of query rows over a paged cache or packed keys (chunks of new tokens, prompts, cross attention), head_dim 128, gfx950, and the
// entry point of the family (argument checks, choice of kernel and of the split of the key axis).
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys row i sees.
//
// Bound: the matrix pipe (4 * 128 FLOP per visible pair and head).  The frame is attn_w16's: a workgroup is 256 rows of one head, four waves of 64 rows,
// ONE wave per SIMD with the whole register file; 128-key stages of K and V in a two-deep LDS ring filled by LDS-DMA behind one barrier per stage; inside a
// wave the step is software-pipelined (matrix stream: P V of sub-tile t-1, then K Q^T of sub-tile t+1; vector stream: softmax of sub-tile t, two
// instructions behind each MFMA); softmax against a fixed reference, the row maximum of the first sub-tile, rows whose sum leaves [2^-60, 2^90) redone
// exactly; row sums on the matrix pipe (a ninth block of ones).  What is different here:
//   * K and V stay row-major in their pages.  V^T fragments come out of LDS through ds_read_b64_tr_b16 (four keys of one column per lane and read), in the
//     key order that the S^T registers have anyway: no transposed copy of V in the cache, no pass that makes one, and K rows in natural order.
//   * addresses: the walk is cut into 16-key groups, which never straddle a page.  64 groups (eight stages) at a time, lane i holds group i's offset
//     (in 16-byte units) and its record count; a DMA piece takes its group's pair with two v_readlane and builds its descriptor in scalar registers, so
//     the page table costs the vector stream next to nothing.  V(s) is issued one stage after K(s) and re-uses K(s)'s pair from scalar registers.
//     The record count cuts the group at the last key that any row sees, and is 0 for a page outside the pool: those rows arrive as zeros.
//   * masks: sub-tiles that every row of the workgroup sees whole run a loop without a mask; the few at the edges of the window, at the sinks and on the
//     diagonal run the same step with one.
//   * the batch is packed: a workgroup finds its request from cu_q by a prefix sum over the lanes.
// Measured (12 heads; by card and clock): 4680 rows over 32 760 keys 793 .. 865 us = 1.09 .. 1.19 PFLOP/s (a large matrix product: 1.32), 0.60 of the cycles of the resident waves in the
// matrix pipe, 228 of 256 compute units busy (19 blocks of 256 rows x 12); a pair of sub-tiles takes 7200 cycles, 4570 of them MFMA, and without the softmax
// 5640, without the DMA 5970, without the LDS fragment reads 6470.  Four rollouts with a window of 9360 keys and 1560 sinks 390 .. 411 us = 0.90 .. 0.95 PFLOP/s, causal prompts of
// ragged requests, 16 heads on 4, 287 .. 298 us = 0.82 .. 0.85, 3 x 4680 rows over 512 text keys 72 us = 0.61 (set-up, first loads and store are half of a four-stage walk).
// Rounding: scores, sums and O in fp32; P to bf16 for the product with V (the matrix operand's type; the sum is taken of the rounded values, so the
// weights add up to one); o once.
#include "attn_ragged.h"
#include "gemm_common.h"

int fvk_attn_rows_launch(const fvk_ragged_args* a, int qb, long row_blocks, int n_split, float* o_part, float* lse_part, hipStream_t s);
int fvk_ragged_merge_launch(const fvk_ragged_args* a, int n_split, float* o_part, float* lse_part, hipStream_t s);

namespace {

using namespace fvk;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int BMQ = RAGGED_BLOCK;
constexpr int KT = 128;              // keys per stage
constexpr int TILE = KT * 256;       // one stage of K or V
constexpr int V_BASE = 2 * TILE;
constexpr int LDS_BYTES = 4 * TILE;  // 131 072
constexpr float L_HIGH = 1.2379400392853803e27f;  // 2^90
constexpr float L_LOW = 8.673617379884035e-19f;   // 2^-60


__device__ __forceinline__ int wave_most(int v) {
    for (int o = 32; o > 0; o >>= 1) {
        const int u = __shfl_xor(v, o, 64);
        v = u > v ? u : v;
    }
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_least(int v) { return -wave_most(-v); }

// query blocks of the batch
template <bool PAGED>
__device__ __forceinline__ int total_blocks(const fvk_ragged_args& a) {
    int n = 0;
    for (int i = threadIdx.x & 63; i < a.R; i += 64) n += (ragged_req<PAGED>(a, i).nq + BMQ - 1) / BMQ;
    return wave_total(n);
}

// what the masks of a workgroup need (wave-uniform)
struct Edges {
    int causal, window, sink, p0;  // p0: place of this wave's first row (causal), else the common place
    RaggedKeys ks;
};

struct Wave {
    bf16x8 qf[4][4];     // Q fragments [q block][k-step of 32 d] (accumulator file)
    f32x4 o[4][9];       // O^T [q block][16-row d block]; block 8: the row sums
    f32x4 s[2][4][4];    // S^T [sub-tile parity][q block][16-key tile]
    u32x4 pf[2][4][2];   // P^T, packed bf16 pairs [sub-tile parity][q block][32-key group]
    bf16x8 ones;
    float mc[4];         // softmax reference * c2, per q block
    int fk[4], fv[8];    // LDS offsets of K fragments [k-step] and V fragments [d block], ring slot included: V of stage j, K of stage j + 1
    float c2;
    unsigned kvo, vvo;   // this lane's source offset inside a group of K / V
    int grp_off, grp_rec;           // lane i: group i of the current eight stages (offset in 16-byte units, valid rows)
    int sv_off[8], sv_rec[8];       // the groups of the stage whose V is issued next (scalar registers)
    const unsigned char *kb, *vb;
    int pdst, zstage, zrows, lane_row;

    // piece I of K(st): group I's rows; keeps the pair for V
    __device__ __forceinline__ void issue_k(int I, int st, int slot) {
        const int at = (st & 7) * 8 + I;
        const int off = __builtin_amdgcn_readlane(grp_off, at), rec = __builtin_amdgcn_readlane(grp_rec, at);
        sv_off[I] = off;
        sv_rec[I] = rec;
        ragged_dma(kb, off, rec, kvo, pdst + slot * TILE, I * 4096);
    }
    // piece I of V(st) from the kept pair; rows below the first key that anybody sees arrive as zeros (they may hold anything)
    __device__ __forceinline__ void issue_v(int I, int st, int slot) {
        unsigned at = vvo;
        if (I == 0) at = lane_row < (st == zstage ? zrows : 0) ? RAGGED_OUT : vvo;
        ragged_dma(vb, sv_off[I], sv_rec[I], at, pdst + slot * TILE, V_BASE + I * 4096);
    }
    __device__ __forceinline__ bf16x8 frag_v(int hf, int G, int db, bool flip = false) const {
        const ragged_lds_byte* at = (const ragged_lds_byte*)(uintptr_t)(unsigned)(fv[db] ^ (flip ? TILE : 0)) + (64 * hf + 32 * G) * 256;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ragged_lds_s16x4*)at);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ragged_lds_s16x4*)(at + 16 * 256));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ bf16x8 frag_k(int ks, int hf, int T, bool flip = false) const {
        return *(const ragged_lds_bf16x8*)((const ragged_lds_byte*)(uintptr_t)(unsigned)(fk[ks] ^ (flip ? TILE : 0)) + (64 * hf + 16 * T) * 256);
    }
    __device__ __forceinline__ void flip_slots() {
#pragma unroll
        for (int c = 0; c < 4; ++c) fk[c] ^= TILE;
#pragma unroll
        for (int c = 0; c < 8; ++c) fv[c] ^= TILE;
    }
    // MFMA result -> compiler-generated reader, and VALU / v_accvgpr_write -> MFMA operand: asm statements get no hazard padding
    template <int PAR>
    __device__ __forceinline__ void fence_s() {
        asm volatile("s_nop 15\n\ts_nop 3"
                     : "+v"(s[PAR][0][0]), "+v"(s[PAR][0][1]), "+v"(s[PAR][0][2]), "+v"(s[PAR][0][3]), "+v"(s[PAR][1][0]), "+v"(s[PAR][1][1]),
                       "+v"(s[PAR][1][2]), "+v"(s[PAR][1][3]), "+v"(s[PAR][2][0]), "+v"(s[PAR][2][1]), "+v"(s[PAR][2][2]), "+v"(s[PAR][2][3]));
        asm volatile("" : "+v"(s[PAR][3][0]), "+v"(s[PAR][3][1]), "+v"(s[PAR][3][2]), "+v"(s[PAR][3][3]));
    }
    __device__ __forceinline__ void fence_o() {
        asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");
#pragma unroll
        for (int qb = 0; qb < 4; ++qb)
            asm volatile("" : "+a"(o[qb][0]), "+a"(o[qb][1]), "+a"(o[qb][2]), "+a"(o[qb][3]), "+a"(o[qb][4]), "+a"(o[qb][5]), "+a"(o[qb][6]), "+a"(o[qb][7]), "+a"(o[qb][8]));
    }
    template <int PAR>
    __device__ __forceinline__ void pv_plain(int hf, bool flip) {
#pragma unroll
        for (int G = 0; G < 2; ++G)
#pragma unroll
            for (int db = 0; db < 9; ++db) {
                const bf16x8 fr = db < 8 ? frag_v(hf, G, db, flip) : ones;
                asm volatile("v_mfma_f32_16x16x32_bf16 %0, %4, %5, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %4, %6, %1\n\t"
                             "v_mfma_f32_16x16x32_bf16 %2, %4, %7, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %4, %8, %3"
                             : "+a"(o[0][db]), "+a"(o[1][db]), "+a"(o[2][db]), "+a"(o[3][db])
                             : "v"(fr), "v"(pf[PAR][0][G]), "v"(pf[PAR][1][G]), "v"(pf[PAR][2][G]), "v"(pf[PAR][3][G]));
            }
    }
    template <int PAR>
    __device__ __forceinline__ void qk_plain(int hf, bool flip) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                const bf16x8 fr = frag_k(ks, hf, T, flip);
                if (ks == 0)
                    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %4, %5, 0\n\tv_mfma_f32_16x16x32_bf16 %1, %4, %6, 0\n\t"
                                 "v_mfma_f32_16x16x32_bf16 %2, %4, %7, 0\n\tv_mfma_f32_16x16x32_bf16 %3, %4, %8, 0"
                                 : "=&v"(s[PAR][0][T]), "=&v"(s[PAR][1][T]), "=&v"(s[PAR][2][T]), "=&v"(s[PAR][3][T])
                                 : "v"(fr), "a"(qf[0][ks]), "a"(qf[1][ks]), "a"(qf[2][ks]), "a"(qf[3][ks]));
                else
                    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %4, %5, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %4, %6, %1\n\t"
                                 "v_mfma_f32_16x16x32_bf16 %2, %4, %7, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %4, %8, %3"
                                 : "+v"(s[PAR][0][T]), "+v"(s[PAR][1][T]), "+v"(s[PAR][2][T]), "+v"(s[PAR][3][T])
                                 : "v"(fr), "a"(qf[0][ks]), "a"(qf[1][ks]), "a"(qf[2][ks]), "a"(qf[3][ks]));
            }
        fence_s<PAR>();
    }
    // scores of keys that their row does not see become -inf: sub-tile t (64 keys) of the walk
    template <int PAR>
    __device__ __forceinline__ void mask(const Edges& e, int t) {
        const int st = t >> 1;
        const int k0 = ragged_stage<KT>(e.ks, st) + 64 * (t & 1);
        const int kmin = st < e.ks.n_sink ? 0 : e.ks.lo, kmax = st < e.ks.n_sink ? e.ks.sink_end : e.ks.hi;
        const int l15 = threadIdx.x & 15, at = k0 + 4 * ((threadIdx.x >> 4) & 3);
        if (e.window == 0) {  // only an upper bound: two instructions per score
#pragma unroll
            for (int qb = 0; qb < 4; ++qb) {
                const int place = e.causal ? e.p0 + 16 * qb + l15 : e.p0;
                const int last = (place + 1 < kmax ? place + 1 : kmax) - at;
#pragma unroll
                for (int T = 0; T < 4; ++T)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[PAR][qb][T][x] = 16 * T + x < last ? s[PAR][qb][T][x] : -INFINITY;
            }
            return;
        }
#pragma unroll
        for (int qb = 0; qb < 4; ++qb) {
            const int place = e.causal ? e.p0 + 16 * qb + l15 : e.p0;
            int first = e.window > 0 ? place - e.window + 1 : kmin;
            first = first > kmin ? first : kmin;
            const int last = (place + 1 < kmax ? place + 1 : kmax) - at, sinks = (st < e.ks.n_sink ? kmax : e.sink) - at;
            first -= at;
            const int low = kmin - at;
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int key = 16 * T + x;
                    const int see = (int)(key < last) & ((int)(key >= first) | (int)(key < sinks)) & (int)(key >= low);
                    s[PAR][qb][T][x] = see ? s[PAR][qb][T][x] : -INFINITY;
                }
        }
    }
    template <int PAR, int QB>
    __device__ __forceinline__ float row_max() const {
        float mx = s[PAR][QB][0][0];
#pragma unroll
        for (int T = 0; T < 4; ++T)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[PAR][QB][T][e]);
        return ragged_max4(mx);
    }
    template <int PAR, int QB>
    __device__ __forceinline__ void exp_pack() {
#pragma unroll
        for (int G = 0; G < 2; ++G)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                bf16x2 p;
#pragma unroll
                for (int y = 0; y < 2; ++y) p[y] = (bf16_t)__builtin_amdgcn_exp2f(__builtin_fmaf(s[PAR][QB][2 * G + (x >> 1)][2 * (x & 1) + y], c2, -mc[QB]));
                pf[PAR][QB][G][x] = __builtin_bit_cast(unsigned, p);
            }
    }
    template <int PAR>
    __device__ __forceinline__ void exp_pack_all() {
        exp_pack<PAR, 0>();
        exp_pack<PAR, 1>();
        exp_pack<PAR, 2>();
        exp_pack<PAR, 3>();
    }
    // the reference from the first sub-tile; a row that sees none of its keys takes 0 (any reference gives the same quotient while the sum stays in range)
    template <int QB>
    __device__ __forceinline__ void reference() {
        const float mx = row_max<0, QB>();
        mc[QB] = mx == -INFINITY ? 0.f : mx * c2;
    }
    // exact online-softmax step: new running maximum first, O and the row sums rescaled
    template <int QB>
    __device__ __forceinline__ void rescale(float mx) {
        const float m_new = fmaxf(mc[QB], mx * c2);
        const float alpha = __builtin_amdgcn_exp2f(mc[QB] - m_new);
#pragma unroll
        for (int d = 0; d < 9; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[QB][d][r] *= alpha;
        mc[QB] = m_new;
    }

    // One step of the pipeline.  Iteration t = 2j + 1 + EVEN of pair j: P V of sub-tile t-1 (V stage j, half EVEN), then K Q^T of sub-tile t+1 (K stage
    // j + 1, half EVEN); the vector stream is the softmax of sub-tile t.  LDS fragments are read FD ahead, each feeds four MFMAs; EVEN = 0 issues the
    // set {K(j+2), V(j+1)}, one piece every eighth MFMA.  The first step has no P V (and K in the other slot), the last one no K Q^T.
    // Empty asm statements that READ a chunk's values keep its work in the chunk.  (As in-out operands they cost a padding s_nop in front of every reader;
    // the loop without masks has 1010 instructions a pair, 272 of them MFMAs.)
    template <int EVEN, bool MASK, bool PV = true, bool QK = true>
    __device__ __forceinline__ void iter(const Edges& e, int st0, int j) {
        constexpr int CUR = 1 - EVEN, FD = 6, PVS = PV ? 18 : 0, SLOTS = PVS + (QK ? 16 : 0), FRAGS = (PV ? 16 : 0) + (QK ? 16 : 0);
        constexpr int STEP = PV && QK ? 2 : 1;  // MFMAs per score
        if (MASK) {
            fence_s<CUR>();
            mask<CUR>(e, 2 * (st0 + j) + 1 + EVEN);
        }
        auto load_frag = [&](int L) {
            const int M = L - (PV ? 16 : 0);
            return M < 0 ? frag_v(EVEN, L >> 3, L & 7) : frag_k(M >> 2, EVEN, M & 3, !PV);
        };
        bf16x8 fr[FD];
#pragma unroll
        for (int i = 0; i < FD; ++i) fr[i] = load_frag(i);
        float ex, p[2];  // exponent of the score after the next one; probabilities of a pair of scores
        p[0] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[CUR][0][0][0], c2, -mc[0]));
        ex = __builtin_fmaf(s[CUR][0][0][1], c2, -mc[0]);
        // operand slots x 4 q blocks: 0-7 V(G = 0), 8 row sums, 9-16 V(G = 1), 17 row sums, then 16 of K
#pragma unroll
        for (int m = 0; m < 4 * SLOTS; ++m) {
            const int F = m >> 2, qb = m & 3;
            const bool is_ones = F < PVS && (F == 8 || F == 17);
            const int L = F >= PVS ? F - (PV ? 2 : 0) : F < 8 ? F : F - 1;
            if (F < PVS) {
                const int G = F >= 9, db = is_ones ? 8 : (F - 9 * G);
                if (is_ones) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(o[qb][8]) : "v"(ones), "v"(pf[EVEN][qb][G]));
                else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(o[qb][db]) : "v"(fr[L % FD]), "v"(pf[EVEN][qb][G]));
            } else {
                const int ks = (F - PVS) >> 2, T = (F - PVS) & 3;
                if (ks == 0) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(s[EVEN][qb][T]) : "v"(fr[L % FD]), "a"(qf[qb][ks]));
                else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(s[EVEN][qb][T]) : "v"(fr[L % FD]), "a"(qf[qb][ks]));
            }
            __builtin_amdgcn_sched_barrier(0);
            if (qb == 3 && !is_ones && L + FD < FRAGS) fr[L % FD] = load_frag(L + FD);
            if (PV && QK && EVEN == 0 && (m & 7) == 1 && m < 128) {  // V first: its pair is overwritten by K's
                const int I = m >> 4;
                if ((m & 8) == 0) issue_v(I, j + 1, (j + 1) & 1);
                else issue_k(I, j + 2, j & 1);
            }
            const int c = m / STEP;
            if (c < 64) {
                if (STEP == 1 || (m & 1) == 0) {
                    if (c & 1) {
                        bf16x2 two;
                        two[0] = (bf16_t)p[0];
                        two[1] = (bf16_t)p[1];
                        pf[CUR][c >> 4][(c >> 3) & 1][(c & 7) >> 1] = __builtin_bit_cast(unsigned, two);
                        asm volatile("" ::"v"(pf[CUR][c >> 4][(c >> 3) & 1][(c & 7) >> 1]));
                    }
                }
                if (STEP == 1 || (m & 1) == 1) {
                    if (c + 1 < 64) p[(c + 1) & 1] = __builtin_amdgcn_exp2f(ex);
                    if (c + 2 < 64) {
                        const int y = c + 2, q_ = y >> 4, x = y & 15;
                        ex = __builtin_fmaf(s[CUR][q_][x >> 2][x & 3], c2, -mc[q_]);
                    }
                    asm volatile("" ::"v"(p[(c + 1) & 1]), "v"(ex));
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// The groups of eight stages from `first` on, one per lane: page-table entry (a load), then offset and records.
template <bool PAGED>
struct Groups : RaggedGroups {
    const int32_t* row;

    __device__ __forceinline__ int load(const RaggedKeys& ks, int first) const {
        if (!PAGED) return 0;
        const int lane = threadIdx.x & 63, st = first + (lane >> 3), k = key<KT>(ks, st, lane & 7);
        const bool in = in_table(st, k);
        return in ? row[in ? k >> shift : 0] : -1;
    }
    __device__ __forceinline__ void set(const RaggedKeys& ks, int first, int page, int& off, int& rec) const {
        const int lane = threadIdx.x & 63, st = first + (lane >> 3);
        const RaggedGroup g = at<PAGED>(ks, st, key<KT>(ks, st, lane & 7), page);
        off = g.off;
        rec = g.rec;
    }
};

template <bool PAGED>
__global__ __launch_bounds__(256, 1) void attn_ragged_kernel(fvk_ragged_args a, RaggedParts part) {
#if defined(__HIP_DEVICE_COMPILE__)
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    FVK_CLAIM_WHOLE_REGISTER_FILE();
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    RaggedReq mine = {0, 0, 0, 0};  // up to 64 requests: request `lane`
    int blocks = 0, total;
    const bool few = a.R <= 64;
    if (few) {
        if (lane < a.R) mine = ragged_req<PAGED>(a, lane);
        blocks = (mine.nq + BMQ - 1) / BMQ;
        total = wave_total(blocks);
    } else {
        total = total_blocks<PAGED>(a);
    }
    const RaggedDeal deal = ragged_deal(a, total, part.n, blockIdx.x);
    if (deal.rank < 0) return;
    const int run = deal.run, h = deal.h, G = a.H / a.Hkv;
    int rank = deal.rank;
    int r = -1, index = 0;
    if (few) {
        RaggedCost cost;  // longest walks first
        cost.init<KT>(a, mine);
        auto at_least = [&](int t) { return cost.at_least(t); };
        int lo = wave_least(cost.least()), hi = wave_most(cost.most()) + 1;
        while (hi - lo > 1) {  // the cost of the block of this rank: the largest t with more than `rank` blocks of t or more
            const int mid = lo + ((hi - lo) >> 1);
            if (wave_total(at_least(mid)) > rank) lo = mid;
            else hi = mid;
        }
        const int above = at_least(lo + 1), same = at_least(lo) - above;
        rank -= wave_total(above);
        const int upto = wave_scan(same);
        const int at = __ffsll(__ballot(upto > rank)) - 1;
        r = at;
        index = __builtin_amdgcn_readlane(blocks - 1 - above, at) - (rank - __builtin_amdgcn_readlane(upto - same, at));
    } else {
        // many requests: in their own order, prefix sums of the block counts, 64 requests at a time
        for (int r0 = 0; r0 < a.R; r0 += 64) {
            const int i = r0 + lane;
            blocks = 0;
            if (i < a.R) blocks = (ragged_req<PAGED>(a, i).nq + BMQ - 1) / BMQ;
            const int upto = wave_scan(blocks);
            const unsigned long long over = __ballot(upto > rank);
            if (over) {
                const int at = __ffsll(over) - 1;
                r = r0 + at;
                index = rank - __builtin_amdgcn_readlane(upto - blocks, at);
                break;
            }
            rank -= __builtin_amdgcn_readlane(upto, 63);
        }
        if (r < 0) return;
    }
    r = __builtin_amdgcn_readfirstlane(r);
    RaggedReq rq;
    if (few) {
        rq.q0 = __builtin_amdgcn_readlane(mine.q0, r);
        rq.nq = __builtin_amdgcn_readlane(mine.nq, r);
        rq.k0 = __builtin_amdgcn_readlane(mine.k0, r);
        rq.len = __builtin_amdgcn_readlane(mine.len, r);
    } else {
        rq = ragged_req<PAGED>(a, r);
    }
    const int first_row = index * BMQ;
    const int last_row = first_row + BMQ < rq.nq ? first_row + BMQ - 1 : rq.nq - 1;
    const RaggedKeys ks = ragged_keys<KT>(a, rq, first_row, last_row);
    const int st0 = (int)((long)ks.n * run / part.n), st1 = (int)((long)ks.n * (run + 1) / part.n);
    const int n = st1 - st0;
    const int row0 = first_row + wave * 64;
    const int kvh = h / G;
    bf16_t* op = (bf16_t*)a.o + (long)rq.q0 * a.o_ts + (long)h * a.o_hs;
    if (n <= 0) {  // no key for any row of this workgroup
        const int row = first_row + tid;
        if (row <= last_row) {
            if (part.n > 1) part.lse[((long)run * a.T + rq.q0 + row) * a.H + h] = -INFINITY;
            else {
                for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(op + (long)row * a.o_ts + c * 8) = make_uint4(0, 0, 0, 0);
                if (a.lse) a.lse[(long)h * a.T + rq.q0 + row] = -INFINITY;
            }
        }
        return;
    }

    Wave w;
    w.c2 = a.scale * 1.4426950408889634f;
    int qrow[4];
    bool q_ok[4];
#pragma unroll
    for (int qb = 0; qb < 4; ++qb) {
        const int row = row0 + 16 * qb + l15;
        q_ok[qb] = row <= last_row;
        qrow[qb] = q_ok[qb] ? row : last_row;
        const bf16_t* qp = (const bf16_t*)a.q + (long)(rq.q0 + qrow[qb]) * a.q_ts + (long)h * a.q_hs;
        // in front of the first LDS-DMA piece, so that they arrive behind the set-up
#pragma unroll
        for (int c = 0; c < 4; ++c) w.qf[qb][c] = ld_bf16x8(qp + c * 32 + g * 8);
    }
    Edges e;
    e.causal = a.causal;
    e.window = a.window;
    e.sink = a.sink;
    e.p0 = a.causal ? rq.len - rq.nq + row0 : rq.len - 1;
    e.ks = ks;
    w.kb = (const unsigned char*)a.k + 2 * (long)kvh * a.k_hs;
    w.vb = (const unsigned char*)a.v + 2 * (long)kvh * a.v_hs;
    w.lane_row = 4 * wave + g;
    const unsigned rs2 = (unsigned)(2 * a.k_rs);
    w.kvo = (unsigned)w.lane_row * rs2 + (unsigned)((l15 ^ w.lane_row) << 4);
    w.vvo = (unsigned)w.lane_row * rs2 + (unsigned)((l15 ^ ((w.lane_row & 7) << 1)) << 4);
    const int lds0 = (int)ragged_lds(smem);  // a multiple of 256 below TILE: the ring's XORs stay inside it
    w.pdst = lds0 + wave * 1024;
    w.zstage = ks.n_sink - st0;
    w.zrows = ks.lo - ks.lo16;
    Groups<PAGED> grp;
    grp.init(a, rq, st1, PAGED);
    grp.row = PAGED ? a.block_table + (long)r * a.table_width : nullptr;
    grp.set(ks, st0, grp.load(ks, st0), w.grp_off, w.grp_rec);
#define WAIT_ALL() asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#define BAR()                                   \
    {                                           \
        __builtin_amdgcn_sched_barrier(0);      \
        __builtin_amdgcn_s_barrier();           \
        __builtin_amdgcn_sched_barrier(0);      \
    }
    // ---- prologue: K(0), V(0) -> slot 0, K(1) -> slot 1; then K Q^T(0), reference, and softmax(0) behind K Q^T(1)
#pragma unroll
    for (int i = 0; i < 8; ++i) w.issue_k(i, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        w.issue_v(i, 0, 0);
        w.issue_k(i, 1, 1);
    }
    int next_page = grp.load(ks, st0 + 8);
    // LDS images: K row x holds its 16-byte chunk c at c ^ (x & 15), V row x its 32-byte piece at piece ^ (x & 7).  Fragments: K row l15 of a 16-key tile;
    // V: lane l15 of group g points at key 4g + l15 / 4, columns 16 db + 4 (l15 % 4)
    const int vrow = 4 * g + (l15 >> 2);
#pragma unroll
    for (int c = 0; c < 4; ++c) w.fk[c] = lds0 + TILE + l15 * 256 + (((4 * c + g) ^ l15) << 4);
#pragma unroll
    for (int c = 0; c < 8; ++c) w.fv[c] = lds0 + V_BASE + vrow * 256 + ((32 * c + 8 * (l15 & 3)) ^ ((vrow & 7) << 5));
#pragma unroll
    for (int qb = 0; qb < 4; ++qb)
#pragma unroll
        for (int d = 0; d < 9; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) w.o[qb][d][x] = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) w.ones[x] = (bf16_t)1.0f;
    asm volatile("" : "+v"(w.ones));  // opaque: a re-materialised constant in front of the asm MFMA that reads it would be an unpadded hazard
    // sub-tiles [ta, tb) of this workgroup's walk are seen whole by all its rows
    int ta, tb;
    {
        const int from = ks.full_lo > ks.lo ? ks.full_lo : ks.lo, to = ks.full_hi < ks.hi ? ks.full_hi : ks.hi;
        ta = 2 * (ks.n_sink - st0) + (from > ks.lo16 ? (from - ks.lo16 + 63) / 64 : 0);
        tb = 2 * (ks.n_sink - st0) + (to > ks.lo16 ? (to - ks.lo16) / 64 : 0);
    }
    // Q into the accumulator file: a use that the compiler waits for (an asm load's register counts as written at once, and may be copied or spilled before
    // it is); the fence behind it pads these writes against the first MFMA
#pragma unroll
    for (int qb = 0; qb < 4; ++qb) asm volatile("" : "+a"(w.qf[qb][0]), "+a"(w.qf[qb][1]), "+a"(w.qf[qb][2]), "+a"(w.qf[qb][3]));
    w.fence_o();
    WAIT_ALL()
    BAR()
    w.template qk_plain<0>(0, true);  // stage 0: the slot fk does not point at
    if (ta > 0 || tb <= 0) w.template mask<0>(e, 2 * st0);
    w.template reference<0>();
    w.template reference<1>();
    w.template reference<2>();
    w.template reference<3>();
    w.template iter<1, false, false, true>(e, st0, -1);
    // ---- pairs j = 0 .. n-2 (sub-tiles 2j+1 and 2j+2): [0, u0) and [u1, n-1) with masks, [u0, u1) seen whole by every row of the workgroup
    const int u0 = clamp_i(ta >> 1, 0, n - 1), u1 = clamp_i((tb - 1) >> 1, u0, n - 1);
    auto head = [&](int j) {
        WAIT_ALL()  // this wave's pieces of the last set have landed
        BAR()       // every wave is past the iteration before: the slots of K(j) and V(j-1) are free
        const int st = j + 2;
        if ((st & 7) == 0) {  // the next eight stages' groups from the page ids loaded eight stages ago
            grp.set(ks, st0 + st, next_page, w.grp_off, w.grp_rec);
            next_page = grp.load(ks, st0 + st + 8);
        }
    };
    int j = 0;
    for (; j < u0; ++j) {
        head(j);
        w.template iter<0, true>(e, st0, j);
        w.template iter<1, true>(e, st0, j);
        w.flip_slots();
    }
    for (; j < u1; ++j) {
        head(j);
        w.template iter<0, false>(e, st0, j);
        w.template iter<1, false>(e, st0, j);
        w.flip_slots();
    }
    for (; j < n - 1; ++j) {
        head(j);
        w.template iter<0, true>(e, st0, j);
        w.template iter<1, true>(e, st0, j);
        w.flip_slots();
    }
    // ---- tail: P V(2n-2), softmax of sub-tile 2n-1, P V(2n-1)
    WAIT_ALL()
    BAR()
    w.template fence_s<1>();
    const int last = 2 * n - 1;
    if (last < ta || last >= tb) w.template mask<1>(e, 2 * st0 + last);
    w.template iter<0, false, true, false>(e, st0, n - 1);
    w.template pv_plain<1>(1, false);
    w.fence_o();
    WAIT_ALL()
    // ---- epilogue: a row whose sum left the safe range is redone exactly and stored again: per row, so that no row's result depends on its neighbours.
    // Lane (l15, g) holds columns 16 d + 4 g + {0..3} of its row.
    bool redo[4];
    {
        const int sink_from = st0 * KT, win_from = st0 > ks.n_sink ? ragged_stage<KT>(ks, st0) : ks.lo, win_to = st1 > ks.n_sink ? ragged_stage<KT>(ks, st1 - 1) + KT : 0;
        const int to = win_to < ks.hi ? win_to : ks.hi, sink_to = ks.sink_end < st1 * KT ? ks.sink_end : st1 * KT;
#pragma unroll
        for (int qb = 0; qb < 4; ++qb) {
            const int place = e.causal ? e.p0 + 16 * qb + l15 : e.p0;
            int first = a.window > 0 && place - a.window + 1 > win_from ? place - a.window + 1 : win_from;
            if (win_from < a.sink) first = win_from;
            const int last = place + 1 < to ? place + 1 : to, last_sink = place + 1 < sink_to ? place + 1 : sink_to;
            const bool sees = first < last || sink_from < last_sink;  // some key of this workgroup's part of the walk
            const float l = w.o[qb][8][0];
            // P up to 2^90 times a value above 2^37 passes fp32 where the quotient does not.  As bit patterns, so that a NaN counts too (two such
            // products of opposite sign leave one; a maximum of floats drops it): without the sign, Inf and NaN are the patterns from 0x7f800000 on
            unsigned top = 0;
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const unsigned bits = __builtin_bit_cast(unsigned, (float)w.o[qb][d][x]) & 0x7fffffffu;
                    top = bits > top ? bits : top;
                }
            redo[qb] = !(l < L_HIGH) || (l < L_LOW && sees) || ragged_max4(top >= 0x7f800000u ? 1.f : 0.f) > 0.f;
        }
    }
    auto store = [&](bool only_redo) {
#pragma unroll
        for (int qb = 0; qb < 4; ++qb) {
            const float l = w.o[qb][8][0];
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            if (!q_ok[qb] || (only_redo && !redo[qb])) continue;
            const long token = rq.q0 + qrow[qb];
            const float lse = l == 0.f ? -INFINITY : w.mc[qb] + log2f(l);
            if (part.n > 1) {
                const long at = ((long)run * a.T + token) * a.H + h;
#pragma unroll
                for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(part.o + at * 128 + d * 16 + g * 4) = w.o[qb][d] * inv;
                if (g == 0) part.lse[at] = lse;
            } else {
                bf16_t* orow = op + (long)qrow[qb] * a.o_ts;
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    bf16x4 v;
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = (bf16_t)(w.o[qb][d][x] * inv);
                    *reinterpret_cast<bf16x4*>(orow + d * 16 + g * 4) = v;
                }
                if (a.lse && g == 0) a.lse[(long)h * a.T + token] = lse;
            }
        }
    };
    if (part.n > 1) {
        store(false);
    } else {
        // Through LDS (the K slots: nobody reads K any more), so that a row leaves as one 256-byte piece: lane (l15, g) writes 8 bytes of its row, 16-byte
        // chunk c at c ^ l15; then 16 lanes read a row and store it: 6000 cycles where stores of 8 bytes straight from the registers took 8600.
        const int area = lds0 + wave * 16384;
#pragma unroll
        for (int qb = 0; qb < 4; ++qb) {
            const float l = w.o[qb][8][0];
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                bf16x4 v;
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] = (bf16_t)(w.o[qb][d][x] * inv);
                *(ragged_lds_bf16x4*)(uintptr_t)(unsigned)(area + (16 * qb + l15) * 256 + (((2 * d + (g >> 1)) ^ l15) << 4) + 8 * (g & 1)) = v;
            }
            if (a.lse && g == 0 && q_ok[qb]) a.lse[(long)h * a.T + rq.q0 + qrow[qb]] = l == 0.f ? -INFINITY : w.mc[qb] + log2f(l);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int x = 4 * i + g, row = row0 + x;
            const bf16x8 v = *(const ragged_lds_bf16x8*)(uintptr_t)(unsigned)(area + x * 256 + l15 * 16);
            if (row <= last_row) st_bf16x8(op + (long)row * a.o_ts + ((l15 ^ (x & 15)) << 3), v);
        }
    }
    if (__syncthreads_or(redo[0] || redo[1] || redo[2] || redo[3])) {
        // the exact pass, one stage at a time through slot 0 (load, wait, compute): running maximum, O and the sums rescaled
        const bool flip_v = ((n - 1) & 1) != 0, flip_k = (n & 1) != 0;  // fv points at the slot of stage n - 1, fk at the other one
#pragma unroll
        for (int qb = 0; qb < 4; ++qb) {
            w.mc[qb] = -__FLT_MAX__;
#pragma unroll
            for (int d = 0; d < 9; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x) w.o[qb][d][x] = 0.f;
        }
        w.fence_o();
        for (int st = 0; st < n; ++st) {
            BAR()  // every wave has finished reading slot 0
            grp.set(ks, st0 + st, grp.load(ks, st0 + st), w.grp_off, w.grp_rec);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w.issue_k(i, 0, 0);
                w.issue_v(i, st, 0);
            }
            WAIT_ALL()
            BAR()
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                w.template qk_plain<0>(hf, flip_k);
                w.template mask<0>(e, 2 * (st0 + st) + hf);
                const float mx[4] = {w.template row_max<0, 0>(), w.template row_max<0, 1>(), w.template row_max<0, 2>(), w.template row_max<0, 3>()};
                w.fence_o();
                w.template rescale<0>(mx[0]);
                w.template rescale<1>(mx[1]);
                w.template rescale<2>(mx[2]);
                w.template rescale<3>(mx[3]);
                w.template exp_pack_all<0>();
                w.fence_o();
                w.template pv_plain<0>(hf, flip_v);
            }
        }
        w.fence_o();
        store(true);  // (straight from the registers: other waves may still read the ring)
    }
#undef WAIT_ALL
#undef BAR
#endif
}

template <bool PAGED>
int launch_blocks(const fvk_ragged_args* a, const RaggedParts& part, int n_blocks, hipStream_t s) {
    static FvkLdsConfigured configured;
    if (int rc = fvk_config_lds(configured, (const void*)attn_ragged_kernel<PAGED>, LDS_BYTES, "fvk_attn_ragged_bf16 (blocks)")) return rc;
    hipLaunchKernelGGL((attn_ragged_kernel<PAGED>), dim3(ragged_grid(a->H, n_blocks, part.n)), dim3(256), LDS_BYTES, s, *a, part);
    FVK_LAUNCH_CHECK();
    return FVK_OK;
}

struct Choice {
    bool blocks;
    int qb, n_split, n_blocks;
    long row_blocks;  // row tiles of a request, at most
};

// Which kernel, which row tile, and how many parts of the key axis, by the time each would take (us).  The model's numbers were fitted to 442 calls (1 .. 32
// requests of 1 .. 1000 rows, 12, 16 and 40 query heads on 4 .. 40 key heads, 20 .. 16 000 keys, equal and ragged lengths), each timed with every tile and
// 1 .. 64 parts: its choice costs 2 % more than the best of them on average and 1.5 times at worst.  One tile size for all (the smallest that holds a
// request's rows) costs up to 2.1 times the best where short prompts meet a hundred rows: a 64-row tile takes 13 us where 16-row ones, side by side, take 6.
//   rows kernel   `round` for a round of 256 workgroups, `more` of that for a further one; and the larger of
//                 `key` per key of a part (a further round: `again` of that), and the stream of all keys at 8.6 TB/s * c / (c + 12.5) with c key streams in
//                 flight (the 256-MB cache included), 5.4 % more for every further tile of the same keys
//   block kernel  per round 12 + 3 for a full one + 3.05 per 128-key stage
//   parts         3.7 (rows kernel) or 2, and their rows written and read at 3.5 TB/s: all T of them, padding too
struct RowsCost {
    double round, more, key, again;
};
constexpr RowsCost ROWS_COST[3] = {{6.2, 0.67, 0.0137, 0.54}, {10.4, 0.58, 0.0139, 0.91}, {13.5, 1.05, 0.0187, 1.16}};  // 16-, 32-, 64-row tiles

Choice choose(const fvk_ragged_args* a) {
    Choice c{};
    const long max_q = a->max_q > 1 ? a->max_q : 1;
    long max_kv = a->max_kv > 1 ? a->max_kv : 1;
    const long seen = (long)a->window + a->sink + (a->causal ? (max_q < 256 ? max_q : 256) : 0);  // by a run of rows
    if (a->window > 0 && seen < max_kv) max_kv = seen;
    const long G = a->H / a->Hkv, rows = max_q * G;
    const double part_us = (double)a->T * a->H * 1024 / 3.5e6;
    const bool may_split = (long)a->T * a->H <= 0xffffffL;  // the merge kernel's grid (2^32 threads)
    auto least = [](long x, long y) { return x < y ? x : y; };
    // block kernel: 32-bit group offsets (16-byte units) and one descriptor stride for K and V are what its address registers hold
    const long reach = a->block_table ? (a->n_pages > 0 ? a->n_pages - 1L : 0L) * a->k_ps + 256L * a->k_rs : (a->total_k + 1024L) * a->k_rs;
    const long n_blocks = (a->T + 255L) / 256 + a->R - 1;  // the batch's blocks at most, whatever the lengths
    const bool fits = a->k_ps == a->v_ps && a->k_rs == a->v_rs && a->k_ps >= 0 && reach / 8 <= 0xffffffffL && (n_blocks + 8) * a->H <= 0x7fffffL;
    c.n_blocks = (int)n_blocks;
#if FVK_VARIANTS  // the tests' choice: rows of a tile (16, 32, 64; 256: the block kernel) + 1024 * parts
    if (const int forced = tunable(TUNE_ATTN_RAGGED)) {
        const int tile = forced % 1024, most = tile == 256 ? 16 : 64;
        c.blocks = tile == 256 && fits;
        c.qb = tile < 64 ? tile / 16 : 4;
        c.row_blocks = (rows + 16 * c.qb - 1) / (16 * c.qb);
        c.n_split = may_split ? (int)least(forced / 1024, most) : 1;
        return c;
    }
#endif
    double best = 0;
    for (int i = 0; i < 3; ++i) {
        const long tile = 16L << i, blocks = (rows + tile - 1) / tile;
        long tiles = ((long)a->T * G + a->R * tile / 2 + tile - 1) / tile;  // ragged rows: half a tile of every request is empty
        tiles = least(a->R * blocks, tiles > a->R ? tiles : a->R) * a->Hkv;
        const long n_of[8] = {1, 2, 4, 8, 256 / tiles, 512 / tiles, 768 / tiles, 1024 / tiles};
        for (long n : n_of) {
            if (n < 1 || n > 64 || (n > 1 && (!may_split || max_kv < 64 * n))) continue;
            const long wgs = tiles * n, all = (long)a->R * a->Hkv, streams = least(all * n, i < 2 ? 512 : 256);
            // one stage per wave: two workgroups of the smaller tiles share a compute unit
            const double again = ((wgs + 255) / 256 - 1) * (i < 2 && max_kv <= 128 * n ? 0.5 : 1.0);
            // several requests: unequal lengths even out over a few rounds (32 streams of 1500 .. 15 600 keys: 206 us with 1024 workgroups, 278 with 256)
            const double even = a->R == 1 || wgs <= 256 ? 1 : wgs >= 1024 ? 0.82 : 1 - 0.18 * (wgs - 256) / 768;
            const double part = ROWS_COST[i].key * max_kv / n * (1 + again * ROWS_COST[i].again);
            const double stream = all * max_kv * 512.0 * (1 + (tiles > all ? 0.054 * (tiles - all) / all : 0)) * (streams + 12.5) / (8.6e6 * streams);
            const double us = ROWS_COST[i].round * (1 + again * ROWS_COST[i].more) + even * (part > stream ? part : stream) + (n > 1 ? 3.7 + n * part_us : 0);
            if (best > 0 && us >= best) continue;
            best = us;
            c.qb = 1 << i;
            c.row_blocks = blocks;
            c.n_split = (int)n;
        }
    }
    if (!fits) return c;
    const long likely = least(least(a->R * ((max_q + 255) / 256), n_blocks), (a->T + 128L * a->R) / 256 + 1);
    const long stages = (max_kv + 127) / 128;
    for (long m = 1; m <= 16 && (m == 1 || (may_split && stages >= 3 * m && (n_blocks + 8) * a->H * m <= 0x7fffffL)); ++m) {
        const long wgs = likely * a->H * m;
        const double us = ((wgs + 255) / 256) * (12 + (wgs < 256 ? wgs * 3 / 256.0 : 3) + 3.05 * ((stages + m - 1) / m)) + (m > 1 ? 2 + m * part_us : 0);
        if (us < best) {
            best = us;
            c.blocks = true;
            c.n_split = (int)m;
        }
    }
    return c;
}

int check(const fvk_ragged_args* a) {
    FVK_CHECK(a->T >= 0 && a->T <= 0x3fffffff && a->R >= 1 && a->R <= 65535, FVK_ERR_ARG, "fvk_attn_ragged_bf16: T=%d R=%d (1..65535 requests)", a->T, a->R);
    FVK_CHECK(a->H >= 1 && a->Hkv >= 1 && a->H <= 4096 && a->H % a->Hkv == 0, FVK_ERR_ARG, "fvk_attn_ragged_bf16: H=%d must be a multiple of Hkv=%d", a->H, a->Hkv);
    if (a->T == 0) return FVK_OK;
    FVK_CHECK(a->q && a->o && a->cu_q && a->kv_lens && ((a->k && a->v) || (!a->block_table && a->total_k == 0)), FVK_ERR_ARG, "fvk_attn_ragged_bf16: null pointer");
    FVK_CHECK(a->scale > 0.f && a->scale < 1e30f, FVK_ERR_ARG, "fvk_attn_ragged_bf16: scale=%g must be positive", a->scale);
    FVK_CHECK(a->window >= 0 && a->sink >= 0 && (a->window > 0 || a->sink == 0), FVK_ERR_ARG, "fvk_attn_ragged_bf16: window=%d sink=%d (a sink needs a window)", a->window, a->sink);
    FVK_CHECK(((a->q_ts | a->q_hs | a->o_ts | a->o_hs | a->k_ps | a->k_rs | a->k_hs | a->v_ps | a->v_rs | a->v_hs) & 7) == 0, FVK_ERR_ARG,
              "fvk_attn_ragged_bf16: strides must be multiples of 8 elements");
    FVK_CHECK((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->o) & 15) == 0, FVK_ERR_ARG, "fvk_attn_ragged_bf16: pointers must be 16-byte aligned");
    FVK_CHECK(a->k_rs >= 0 && a->v_rs >= 0 && a->k_rs <= (1 << 24) && a->v_rs <= (1 << 24), FVK_ERR_ARG, "fvk_attn_ragged_bf16: row strides %ld, %ld must be at most 2^24 elements", a->k_rs, a->v_rs);
    if (a->block_table) {
        FVK_CHECK(a->page_shift >= 4 && a->page_shift <= 8, FVK_ERR_ARG, "fvk_attn_ragged_bf16: page_size=%d must be 16, 32, 64, 128 or 256", a->page_shift >= 0 && a->page_shift < 31 ? 1 << a->page_shift : -1);
        FVK_CHECK(a->table_width >= 1 && a->n_pages >= 0 && ((long)a->table_width << a->page_shift) <= 0x3fffffffL, FVK_ERR_ARG, "fvk_attn_ragged_bf16: table_width=%d n_pages=%d", a->table_width, a->n_pages);
    } else {
        FVK_CHECK(a->total_k >= 0 && a->total_k <= 0x3fffffff, FVK_ERR_ARG, "fvk_attn_ragged_bf16: total_k=%d", a->total_k);
        FVK_CHECK(!a->causal && a->window == 0, FVK_ERR_ARG, "fvk_attn_ragged_bf16: packed keys (cross attention) take no causal mask and no window");
    }
    return FVK_OK;
}

// The caller's arguments as the kernels take them: the stride of a dimension of one element says nothing (0); a window or sink behind the longest
// possible cache is that length (the kernels subtract them from places).
fvk_ragged_args plain(const fvk_ragged_args* a) {
    fvk_ragged_args b = *a;
    if (b.T == 1) b.q_ts = b.o_ts = 0;
    if (b.H == 1) b.q_hs = b.o_hs = 0;
    if (b.Hkv == 1) b.k_hs = b.v_hs = 0;
    if (!b.block_table || b.n_pages == 1) b.k_ps = b.v_ps = 0;
    if (!b.block_table && b.total_k == 1) b.k_rs = b.v_rs = 0;
    b.window = b.window < 0x3fffffff ? b.window : 0x3fffffff;
    b.sink = b.sink < 0x3fffffff ? b.sink : 0x3fffffff;
    return b;
}

}  // namespace

extern "C" long fvk_attn_ragged_workspace_bytes(const fvk_ragged_args* args) {
    FVK_CHECK(args, -1, "fvk_attn_ragged_workspace_bytes: null args");
    const fvk_ragged_args b = plain(args), *a = &b;
    if (check(a) != FVK_OK) return -1;
    if (a->T == 0) return 0;
    const Choice c = choose(a);
    return c.n_split > 1 ? (long)c.n_split * a->T * a->H * 129 * 4 : 0;
}

extern "C" int fvk_attn_ragged_choice(const fvk_ragged_args* args, int* tile, int* parts) {
    FVK_CHECK(args && tile && parts, FVK_ERR_ARG, "fvk_attn_ragged_choice: null pointer");
    const fvk_ragged_args b = plain(args), *a = &b;
    if (int rc = check(a)) return rc;
    const Choice c = choose(a);
    *tile = c.blocks ? BMQ : 16 * c.qb;
    *parts = c.n_split;
    return FVK_OK;
}

extern "C" int fvk_attn_ragged_bf16(const fvk_ragged_args* args, void* ws, long ws_bytes, void* stream) {
    FVK_CHECK(args, FVK_ERR_ARG, "fvk_attn_ragged_bf16: null args");
    const fvk_ragged_args b = plain(args), *a = &b;
    if (int rc = check(a)) return rc;
    if (a->T == 0) return FVK_OK;
    const Choice c = choose(a);
    const long need = c.n_split > 1 ? (long)c.n_split * a->T * a->H * 129 * 4 : 0;
    FVK_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0), FVK_ERR_ARG, "fvk_attn_ragged_bf16: workspace of %ld bytes, 16-byte aligned, needed (got %ld)", need, ws ? ws_bytes : 0L);
    float* o_part = (float*)ws;
    float* lse_part = o_part + (long)c.n_split * a->T * a->H * 128;
    const RaggedParts part{o_part, lse_part, c.n_split};
    if (c.blocks) {
        if (int rc = a->block_table ? launch_blocks<true>(a, part, c.n_blocks, (hipStream_t)stream) : launch_blocks<false>(a, part, c.n_blocks, (hipStream_t)stream)) return rc;
    } else if (int rc = fvk_attn_rows_launch(a, c.qb, c.row_blocks, c.n_split, o_part, lse_part, (hipStream_t)stream)) return rc;
    return c.n_split > 1 ? fvk_ragged_merge_launch(a, c.n_split, o_part, lse_part, (hipStream_t)stream) : FVK_OK;
}
