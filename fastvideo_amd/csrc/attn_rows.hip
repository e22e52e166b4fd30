// Ragged attention for FEW query rows per request (single tokens, short chunks) over a paged cache or packed keys, head_dim 128, gfx950.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys row i sees, one pass over the keys with a running maximum and sum.
//
// Bound: a row of a single-token step needs 512 B of K and V per key and 4 * 128 FLOP per head — HBM.  So the K / V stream decides everything:
//   * rows of one request that share a key head (its new tokens x the group's query heads) are ONE tile of 16 * QB rows: the key head's pages are
//     read once for all of them, and the matrix pipe does the products (S^T = K Q^T, O^T = V^T P^T with v_mfma_f32_16x16x32_bf16) however few
//     rows are real;
//   * every wave streams its own 32-key stages (K 8 KB + V 8 KB) through a private two-stage LDS ring by LDS-DMA with counted vmcnt; no barrier until the
//     four waves' results are merged.  64 KB in flight per CU.  Where a wave has one stage at most, a ring of one, and two workgroups per CU;
//   * the key axis of a request is cut over workgroups (gridDim.x) as well; their parts are merged by ragged_merge_kernel.
// K rows stay row-major [key][d]: A operand of S^T.  V rows too: ds_read_b64_tr_b16 hands each lane four keys of one column, which is the A operand of O^T,
// so neither the cache nor a pass over it holds a transposed copy.  P^T is the S^T registers of the same lane: lane (q = lane & 15, g = lane >> 4) holds keys
// 4g..4g+3 of each 16-key tile, and the two tr reads of a V fragment fetch exactly those keys.
// LDS images: K row r holds its 16-byte chunk c at c ^ (r & 15), V row r its 32-byte piece at piece ^ (r & 7): every fragment read touches all banks once.
// Measured: one token over 900 keys, 12 heads, 5.9 us and 2.9 for the merge of its parts (launch latency); 32 streams over 1500 .. 15 600 keys, 40 heads on 8,
// 198 us and 4.7 (1.05 GB, 5.1 TB/s; a large copy reaches 4.8); 5 requests of 84 .. 186 rows over 0 .. 47 states, 12 heads, 10.1 us.
// Rounding: scores, maximum, sum and O in fp32; P to bf16 for the product with V (the matrix operand's type; the sum is taken before that rounding, so a
// row's weights add up to one within 2^-8; the block kernel's sum is taken after it); o once.
#include "attn_ragged.h"

namespace {

using namespace fvk;

constexpr int ST = 32;                  // keys per stage
constexpr int STAGE_BYTES = ST * 512;   // K and V
constexpr int O_PITCH = 132;            // floats per row of the merge area: 16 rows apart by 4 banks

constexpr int rows_lds(int qb, int stages) {
    const int ring = 4 * stages * STAGE_BYTES, merge = 4 * 16 * qb * (O_PITCH + 2) * 4;
    return ring > merge ? ring : merge;
}

#if defined(__HIP_DEVICE_COMPILE__)
template <int QB, bool PAGED, int STAGES>
__device__ __forceinline__ void attn_rows(const fvk_ragged_args& a, const RaggedParts& part, int flat) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.y % a.Hkv, rb_step = gridDim.y / a.Hkv;
    const int G = a.H / a.Hkv;
    int r = blockIdx.z, first = blockIdx.y / a.Hkv;
    if (flat) {  // gridDim.z counts the batch's tiles, request after request: no workgroups for tiles that a short request does not have
        int rank = blockIdx.z;
        r = -1;
        for (int r0 = 0; r0 < a.R; r0 += 64) {
            const int i = r0 + lane;
            const int tiles = i < a.R ? (int)(((long)ragged_req<PAGED>(a, i).nq * G + 16 * QB - 1) / (16 * QB)) : 0;
            const int upto = wave_scan(tiles);
            const unsigned long long over = __ballot(upto > rank);
            if (over) {
                const int at = __ffsll(over) - 1;
                r = r0 + at;
                first = rank - __builtin_amdgcn_readlane(upto - tiles, at);
                break;
            }
            rank -= __builtin_amdgcn_readlane(upto, 63);
        }
        if (r < 0) return;  // the host's bound on the number of tiles is not tight
        r = __builtin_amdgcn_readfirstlane(r);
        first = __builtin_amdgcn_readfirstlane(first);
    }
    const RaggedReq rq = ragged_req<PAGED>(a, r);
    const int rows = rq.nq * G;
    const float c2 = a.scale * 1.4426950408889634f;
    const bf16_t* kb = (const bf16_t*)a.k + (long)kvh * a.k_hs + (PAGED ? 0L : (long)rq.k0 * a.k_rs);
    const bf16_t* vb = (const bf16_t*)a.v + (long)kvh * a.v_hs + (PAGED ? 0L : (long)rq.k0 * a.v_rs);
    unsigned char* ring = smem + wave * STAGES * STAGE_BYTES;
    RaggedPages pages;
    if (PAGED) pages.init(a, r);
    // LDS-DMA: instruction i of 16 rows writes rows 4i .. 4i+3 (lane >> 4) linearly, so a lane fetches the chunk that belongs at its place
    unsigned k_off[4], v_off[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) k_off[i] = (unsigned)((4 * i + g) * a.k_rs * 2) + (unsigned)((l15 ^ (4 * i + g)) << 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) v_off[i] = (unsigned)(g * a.v_rs * 2) + (unsigned)((l15 ^ (((4 * i + g) & 7) << 1)) << 4);

    for (int rb = first; rb * 16 * QB < rows; rb += rb_step) {
        const int row0 = rb * 16 * QB, row1 = row0 + 16 * QB < rows ? row0 + 16 * QB : rows;
        const RaggedKeys ks = ragged_keys<ST>(a, rq, row0 / G, (row1 - 1) / G);
        const int st0 = (int)((long)ks.n * blockIdx.x / gridDim.x), st1 = (int)((long)ks.n * (blockIdx.x + 1) / gridDim.x);
        // this lane's rows
        bf16x8 qf[QB][4];
        int place[QB];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const int rho = row0 + 16 * qb + l15 < rows ? row0 + 16 * qb + l15 : rows - 1;
            const int i = rho / G, h = kvh * G + rho - i * G;
            place[qb] = a.causal ? rq.len - rq.nq + i : rq.len - 1;
            const bf16_t* qp = (const bf16_t*)a.q + (long)(rq.q0 + i) * a.q_ts + (long)h * a.q_hs;
#pragma unroll
            for (int s = 0; s < 4; ++s) qf[qb][s] = ld_bf16x8(qp + s * 32 + g * 8);
        }
        // a use in front of the first LDS-DMA: the compiler would wait for these loads inside the loop, and with them for the stage in flight
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) asm volatile("" : "+v"(qf[qb][0]), "+v"(qf[qb][1]), "+v"(qf[qb][2]), "+v"(qf[qb][3]));
        f32x4 o[QB][8];
        float m[QB], l[QB];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            m[qb] = -__FLT_MAX__;
            l[qb] = 0.f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[qb][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        auto issue = [&](int s, int slot) {
            const int k0 = ragged_stage<ST>(ks, s);
            const int kmin = s < ks.n_sink ? 0 : ks.lo, kmax = ragged_end(ks, s);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int key = k0 + 16 * half;
                const RaggedHalf at16 = ragged_half<PAGED>(a, key, kmax, PAGED ? (key < kmax ? pages.get(key >> a.page_shift) : -1) : 0);
                const unsigned dst = ragged_lds(ring) + slot * STAGE_BYTES + half * 4096;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = key + 4 * i + g;
                    const bool in = at >= kmin && at < kmax;
                    ragged_dma((const unsigned char*)(kb + at16.k), 0, at16.k_rec, in ? k_off[i] : RAGGED_OUT, dst + i * 1024);
                    ragged_dma((const unsigned char*)(vb + at16.v), 0, at16.v_rec, in ? v_off[i & 1] + (unsigned)(4 * i * a.v_rs * 2) : RAGGED_OUT, dst + 8192 + i * 1024);
                }
            }
        };

        int s = st0 + wave;
        if (s < st1) issue(s, 0);
        if (STAGES > 1 && s + 4 < st1) issue(s + 4, 1);
        for (int slot = 0; s < st1; s += 4, slot ^= STAGES - 1) {
            if (STAGES > 1 && s + 4 < st1) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");  // the 16 pieces of the next stage may still fly
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            const unsigned char* kl = ring + slot * STAGE_BYTES;
            const unsigned char* vl = kl + 8192;
            f32x4 sc[QB][2];
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) sc[qb][0] = sc[qb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kl + (16 * t + l15) * 256 + (((4 * c + g) ^ l15) << 4));
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) sc[qb][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[qb][c], sc[qb][t], 0, 0, 0);
                }
            const int k0 = ragged_stage<ST>(ks, s);
            const int kmin = s < ks.n_sink ? 0 : ks.lo, kmax = ragged_end(ks, s);
            const bool full = k0 >= kmin && k0 + ST <= kmax && k0 + ST <= ks.full_hi && (s < ks.n_sink || k0 >= ks.full_lo);
            bf16x8 pf[QB];
            bool grew = false;
            float alpha[QB];
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                if (!full) {
                    const int first = a.window > 0 && place[qb] - a.window + 1 > kmin ? place[qb] - a.window + 1 : kmin;
                    const int last = place[qb] + 1 < kmax ? place[qb] + 1 : kmax;
                    const int sinks = s < ks.n_sink ? kmax : a.sink;
                    // selects, no branches: with `&&` / `||` here the compiler built a branch per score and lost the -inf of one of them
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int key = k0 + 16 * (x >> 2) + 4 * g + (x & 3);
                        const bool see = (int)(key < last) & ((int)(key >= first) | (int)(key < sinks)) & (int)(key >= kmin);
                        sc[qb][x >> 2][x & 3] = see ? sc[qb][x >> 2][x & 3] : -INFINITY;
                    }
                }
                float mx = fmaxf(fmaxf(fmaxf(sc[qb][0][0], sc[qb][0][1]), fmaxf(sc[qb][0][2], sc[qb][0][3])),
                                 fmaxf(fmaxf(sc[qb][1][0], sc[qb][1][1]), fmaxf(sc[qb][1][2], sc[qb][1][3])));
                mx = ragged_max4(mx);
                const float m_new = fmaxf(m[qb], mx);
                grew |= m_new > m[qb];
                alpha[qb] = __builtin_amdgcn_exp2f((m[qb] - m_new) * c2);
                m[qb] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const float p = __builtin_amdgcn_exp2f((sc[qb][x >> 2][x & 3] - m_new) * c2);
                    sum += p;
                    pf[qb][x] = (bf16_t)p;
                }
                l[qb] = l[qb] * alpha[qb] + sum;
            }
            if (__any(grew)) {
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int d = 0; d < 8; ++d) o[qb][d] *= alpha[qb];
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                // lane L of a 16-lane group points at key 4g + L / 4, columns 16 d + 4 (L % 4) ..: it receives column 16 d + L of keys 4g .. 4g + 3
                const int row = 4 * g + (l15 >> 2);
                const unsigned char* at = vl + row * 256 + ((32 * d + 8 * (l15 & 3)) ^ ((row & 7) << 5));
                const s16x4 va = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ragged_lds_s16x4*)at);
                const s16x4 vc = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ragged_lds_s16x4*)(at + 16 * 256));  // row + 16: the same swizzle
                const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(va, vc, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) o[qb][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[qb], o[qb][d], 0, 0, 0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
            __builtin_amdgcn_sched_barrier(0);
            if (s + 4 * STAGES < st1) issue(s + 4 * STAGES, slot);
        }

        // ---- merge the four waves: each leaves (O, m, l) of its rows
        __syncthreads();
        float* om = reinterpret_cast<float*>(smem);
        float* ml = om + 4 * 16 * QB * O_PITCH;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            l[qb] += __shfl_xor(l[qb], 16);
            l[qb] += __shfl_xor(l[qb], 32);
            const int row = wave * 16 * QB + 16 * qb + l15;
#pragma unroll
            for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(om + row * O_PITCH + 16 * d + 4 * g) = o[qb][d];
            if (g == 0) {
                ml[2 * row] = m[qb];
                ml[2 * row + 1] = l[qb];
            }
        }
        __syncthreads();
        for (int x = tid; x < 16 * QB * 32; x += 256) {
            const int row = x >> 5, d4 = (x & 31) * 4, rho = row0 + row;
            if (rho >= rows) continue;
            float top = -__FLT_MAX__;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[2 * (w * 16 * QB + row)]);
            float total = 0.f;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int at = w * 16 * QB + row;
                const float weight = __builtin_amdgcn_exp2f((ml[2 * at] - top) * c2);
                total += ml[2 * at + 1] * weight;
                acc += *reinterpret_cast<const f32x4*>(om + at * O_PITCH + d4) * weight;
            }
            const float inv = total == 0.f ? 0.f : 1.0f / total;  // no key seen: zeros
            acc *= inv;
            const int i = rho / G, h = kvh * G + rho - i * G;
            const long token = rq.q0 + i;
            const float lse = total == 0.f ? -INFINITY : top * c2 + log2f(total);
            if (part.n > 1) {
                const long at = ((long)blockIdx.x * a.T + token) * a.H + h;
                *reinterpret_cast<f32x4*>(part.o + at * 128 + d4) = acc;
                if (d4 == 0) part.lse[at] = lse;
            } else {
                bf16x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (bf16_t)acc[e];
                *reinterpret_cast<bf16x4*>((bf16_t*)a.o + token * a.o_ts + (long)h * a.o_hs + d4) = v;
                if (a.lse && d4 == 0) a.lse[(long)h * a.T + token] = lse;
            }
        }
        if (flat) break;
        __syncthreads();
    }
}
#endif

// The two-stage ring: MFMAs while the wave's own LDS-DMA pieces fly, one workgroup per compute unit (128 KB of LDS), so one wave per SIMD: it owns the
// register file (fvk_common.h: FVK_CLAIM_WHOLE_REGISTER_FILE), whatever its 123 .. 471 registers would leave to a neighbour.
template <int QB, bool PAGED>
__global__ __launch_bounds__(256, 1) void attn_rows_ring_kernel(fvk_ragged_args a, RaggedParts part, int flat) {
#if defined(__HIP_DEVICE_COMPILE__)
    FVK_CLAIM_WHOLE_REGISTER_FILE();
    attn_rows<QB, PAGED, 2>(a, part, flat);
#endif
}

// One stage: a wave has waited for all its pieces before its first MFMA.  Two workgroups of the smaller tiles share a compute unit and claim half of the
// register file each; the 64-row tile is alone and claims all of it.
template <int QB, bool PAGED>
__global__ __launch_bounds__(256, QB <= 2 ? 2 : 1) void attn_rows_kernel(fvk_ragged_args a, RaggedParts part, int flat) {
#if defined(__HIP_DEVICE_COMPILE__)
    if (QB <= 2) asm volatile("" ::: "v255");
    else FVK_CLAIM_WHOLE_REGISTER_FILE();
    attn_rows<QB, PAGED, 1>(a, part, flat);
#endif
}

// o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max).  Latency decides (a token's row reads part.n * 512 B), so all parts of a row are in flight at
// once: half a wave holds a part's row (four columns per lane) and reads up to eight parts; WIDE (more than eight parts): the eight half waves of a
// workgroup share one row.  (One part after the other by one wave: 30 us at 64 parts.)  Tokens behind the last request have no parts and stay as they are.
template <bool WIDE>
__global__ __launch_bounds__(256) void ragged_merge_kernel(fvk_ragged_args a, RaggedParts part) {
    __shared__ f32x4 sums[8][32];
    __shared__ float totals[8];
    const int half = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long rows = (long)a.T * a.H, id = WIDE ? (long)blockIdx.x : (long)blockIdx.x * 8 + half;
    const long token = id / a.H;
    const int h = (int)(id - token * a.H);
    const bool real = id < rows && token >= a.cu_q[0] && token < a.cu_q[a.R];
    if (WIDE && !real) return;
    f32x4 v[8];
    float lse[8], top = -INFINITY;
    const int parts = real ? (WIDE ? (part.n - half + 7) / 8 : part.n) : 0;  // this half wave's
    const long step = WIDE ? 8 * rows : rows;
    const float* lp = part.lse + (WIDE ? half * rows : 0) + (real ? id : 0);
    const float* op = part.o + ((WIDE ? half * rows : 0) + (real ? id : 0)) * 128 + lane * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // an absent part's place is taken by the first one's address (every row has one), its weight is 0
        const long at = i < parts ? i * step : 0;
        const bool in = i < parts;
        lse[i] = lp[in ? at : 0];
        v[i] = *reinterpret_cast<const f32x4*>(op + (in ? at * 128 : 0));
        lse[i] = in ? lse[i] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, lse[i]);
    if (WIDE) {
        if (lane == 0) totals[half] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, totals[i]);
        __syncthreads();
    }
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float w = lse[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lse[i] - top);
        total += w;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += lse[i] == -INFINITY ? 0.f : v[i][e] * w;  // a part without keys wrote no row
    }
    if (WIDE) {
        sums[half][lane] = acc;
        if (lane == 0) totals[half] = total;
        __syncthreads();
        if (half > 0) return;
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            acc += sums[i][lane];
            total += totals[i];
        }
    }
    if (!real) return;
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (bf16_t)(acc[e] * inv);
    *reinterpret_cast<bf16x4*>((bf16_t*)a.o + token * a.o_ts + (long)h * a.o_hs + lane * 4) = o;
    if (a.lse && lane == 0) a.lse[(long)h * a.T + token] = total == 0.f ? -INFINITY : top + log2f(total);
}

template <int QB, bool PAGED>
int launch_rows(const fvk_ragged_args* a, const RaggedParts& part, long row_blocks, hipStream_t s) {
    static FvkLdsConfigured one, ring;
    // parts of at most four stages by the host's bound: a ring of one stage, so that two workgroups fit a compute unit
    const int stages = (long)a->max_kv <= 4L * ST * part.n ? 1 : 2;
    if (int rc = stages == 1 ? fvk_config_lds(one, (const void*)attn_rows_kernel<QB, PAGED>, rows_lds(QB, 1), "fvk_attn_ragged_bf16 (rows)")
                             : fvk_config_lds(ring, (const void*)attn_rows_ring_kernel<QB, PAGED>, rows_lds(QB, 2), "fvk_attn_ragged_bf16 (rows)"))
        return rc;
    // several tiles in some request: one workgroup per tile of the batch (at most T * G / tile + R of them), as long as gridDim.z holds them
    const long tiles = (long)a->T * (a->H / a->Hkv) / (16 * QB) + a->R;
    const bool flat = a->R > 1 && row_blocks > 1 && tiles <= 65535;
    const long cap = 65535 / a->Hkv;  // gridDim.y; the kernel walks on where there are more
    const unsigned y = flat ? a->Hkv : (unsigned)(a->Hkv * (row_blocks < cap ? row_blocks : cap));
    const dim3 grid(part.n, y, flat ? (unsigned)tiles : (unsigned)a->R);
    if (stages == 1) hipLaunchKernelGGL((attn_rows_kernel<QB, PAGED>), grid, dim3(256), rows_lds(QB, 1), s, *a, part, (int)flat);
    else hipLaunchKernelGGL((attn_rows_ring_kernel<QB, PAGED>), grid, dim3(256), rows_lds(QB, 2), s, *a, part, (int)flat);
    FVK_LAUNCH_CHECK();
    return FVK_OK;
}

}  // namespace

int fvk_attn_rows_launch(const fvk_ragged_args* a, int qb, long row_blocks, int n_split, float* o_part, float* lse_part, hipStream_t s) {
    const RaggedParts part{o_part, lse_part, n_split};
    if (a->block_table) return qb == 1 ? launch_rows<1, true>(a, part, row_blocks, s) : qb == 2 ? launch_rows<2, true>(a, part, row_blocks, s) : launch_rows<4, true>(a, part, row_blocks, s);
    return qb == 1 ? launch_rows<1, false>(a, part, row_blocks, s) : qb == 2 ? launch_rows<2, false>(a, part, row_blocks, s) : launch_rows<4, false>(a, part, row_blocks, s);
}

int fvk_ragged_merge_launch(const fvk_ragged_args* a, int n_split, float* o_part, float* lse_part, hipStream_t s) {
    const long rows = (long)a->T * a->H;
    const RaggedParts part{o_part, lse_part, n_split};
    if (n_split > 8) hipLaunchKernelGGL((ragged_merge_kernel<true>), dim3((unsigned)rows), dim3(256), 0, s, *a, part);
    else hipLaunchKernelGGL((ragged_merge_kernel<false>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, *a, part);
    FVK_LAUNCH_CHECK();
    return FVK_OK;
}
