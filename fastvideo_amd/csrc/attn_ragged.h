// What the kernels of the ragged attention family share (attn_rows.hip: few rows per request; attn_ragged.hip: blocks of rows): the argument
// block, the key range of a run of rows and the stages that cover it (ragged_walk.h), and the LDS-DMA of 16 key rows from a page (or from packed rows).
//
// The batch is packed: request r owns q rows [cu_q[r], cu_q[r+1]) and either the first kv_lens[r] tokens of its pages (block_table row r) or
// the rows [cu_k[r], cu_k[r+1]) of packed k / v.  Row i of nq rows has the place p = len - 1 (all rows see the whole cache) or
// p = len - nq + i (causal); it sees the keys j <= p with (no window, or j > p - window, or j < sink).
//
// All lengths are read on the GPU and clamped to what the tensors hold: a wrong cu_q, kv_lens or block_table gives wrong numbers, never an access
// outside the tensors.  A page id outside the pool reads as zero rows (its buffer descriptor has no records).
#pragma once
#include "fvk_common.h"
#include "ragged_walk.h"

namespace fvk {

typedef __attribute__((address_space(3))) unsigned char ragged_lds_byte;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 ragged_lds_s16x4;
typedef __attribute__((address_space(3))) bf16x8 ragged_lds_bf16x8;
typedef __attribute__((address_space(3))) bf16x4 ragged_lds_bf16x4;

constexpr unsigned RAGGED_OUT = 0x80000000u;  // a buffer offset past every descriptor: the row arrives as zeros

struct RaggedParts {  // partial results of a split key axis: normalised rows and base-2 log-sum-exp, [split][token][head]
    float* o;
    float* lse;
    int n;
};

// over the 64 lanes, by DPP (a few cycles a step; the shuffles through LDS cost ten times that): inclusive prefix sums and totals
__device__ __forceinline__ int wave_scan(int v) {
#define STEP(CTRL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
    STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf)  // row_shr 1, 2, 4, 8
    STEP(0x142, 0xa) STEP(0x143, 0xc)                                    // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
#undef STEP
    return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
// 1 KB from memory to LDS: 16 bytes per lane from base + 16 * off16 + at (zeros where that passes `records` bytes behind base + 16 * off16), to lds + 16 * lane.
// Written out because a ds_read_b64_tr_b16 behind the builtin makes the compiler wait for ALL loads in flight (vmcnt(0) in front of every V fragment; the
// block kernel ran at half its rate with it): it cannot know that the fragment's ring slot is another one.  The waits are the kernels' own: counted vmcnt.
// It has no register result that could arrive late.  The descriptor goes through scalar moves because a scalar register that a vector instruction
// (v_readlane) wrote may not feed a memory instruction within five wait states, and asm gets no padding.
__device__ __forceinline__ void ragged_dma(const unsigned char* base, unsigned off16, unsigned records, unsigned at, unsigned lds, int lds_more = 0) {
    const unsigned long b = (unsigned long)base;
    asm volatile("s_add_u32 m0, %5, %6\n\t"  // m0: no allocatable register, and nothing here keeps a value in it
                 "s_lshl_b32 s96, %2, 4\n\t"
                 "s_lshr_b32 s97, %2, 28\n\t"
                 "s_add_u32 s96, s96, %0\n\t"
                 "s_addc_u32 s97, s97, %1\n\t"
                 "s_mov_b32 s98, %3\n\t"
                 "s_mov_b32 s99, 0x00020000\n\t"
                 "buffer_load_dwordx4 %4, s[96:99], 0 offen lds"
                 :
                 : "s"((unsigned)b), "s"((unsigned)(b >> 32)), "s"(off16), "s"(records), "v"(at), "s"(lds), "i"(lds_more)
                 : "memory", "scc", "s96", "s97", "s98", "s99");
}
__device__ __forceinline__ unsigned ragged_lds(const unsigned char* p) { return (unsigned)(uintptr_t)(ragged_lds_byte*)p; }

// over the four lanes {l, l ^ 16, l ^ 32, l ^ 48} that share a query row, by lane swaps in the vector pipe
__device__ __forceinline__ float ragged_max4(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned w = __builtin_bit_cast(unsigned, fmaxf(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)b[0]), __builtin_bit_cast(float, (unsigned)b[1]));
}

// Page ids of one request, 64 at a time in a register (lane i: page first + i): an id is one v_readlane away, and the table is read once per 64 pages.
struct RaggedPages {
    const int32_t* row;
    int width, first, ids, n_pages;
    __device__ __forceinline__ void init(const fvk_ragged_args& a, int r) {
        row = a.block_table + (long)r * a.table_width;
        width = a.table_width;
        n_pages = a.n_pages;
        first = -0x40000000;
        ids = -1;
    }
    __device__ __forceinline__ int get(int index) {  // index: the same in all lanes
        if ((unsigned)(index - first) >= 64u) {
            first = index;
            const int at = index + (int)(threadIdx.x & 63);
            ids = at >= 0 && at < width ? row[at] : -1;
        }
        return __builtin_amdgcn_readlane(ids, index - first);
    }
};

}  // namespace fvk
