// Whole-number arithmetic of the ragged attention kernels (attn_rows.hip, attn_ragged.hip): which rows and keys a request has, which workgroup takes which
// block of rows, which stages of keys it walks and where a 16-key group lies in memory.  Host and device: tests/ragged_bounds.cpp runs these very functions
// over random lengths, windows, strides and wrong metadata on the CPU and holds every address against its tensor.
#pragma once
#include "../../include/fvk_amd.h"

#if defined(__HIPCC__)
#define FVK_HD __host__ __device__ __forceinline__
#else
#define FVK_HD inline
#endif

namespace fvk {

constexpr int RAGGED_BLOCK = 256;  // rows of a block kernel's workgroup

FVK_HD int clamp_i(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

struct RaggedReq {
    int q0, nq;  // first row, rows
    int k0, len; // packed keys: first row; keys
};

template <bool PAGED>
FVK_HD RaggedReq ragged_req(const fvk_ragged_args& a, int r) {
    RaggedReq q;
    q.q0 = clamp_i(a.cu_q[r], 0, a.T);
    const int q1 = clamp_i(a.cu_q[r + 1], 0, a.T);
    q.nq = q1 > q.q0 ? q1 - q.q0 : 0;
    if (PAGED) {
        q.k0 = 0;
        q.len = clamp_i(a.kv_lens[r], 0, a.table_width << a.page_shift);
    } else {
        q.k0 = clamp_i(a.kv_lens[r], 0, a.total_k);
        const int k1 = clamp_i(a.kv_lens[r + 1], 0, a.total_k);
        q.len = k1 > q.k0 ? k1 - q.k0 : 0;
    }
    return q;
}

// The keys that some row of the token run [i0, i1] sees, as [0, sink_end) and [lo, hi), in stages of STAGE keys; keys in [full_lo, full_hi) of the
// second part are seen by every row of the run (those of the first part by every row whose place is behind them: full_hi again).
struct RaggedKeys {
    int sink_end, lo, hi, lo16, n_sink, n;  // n stages, the first n_sink of them over [0, sink_end)
    int full_lo, full_hi;
};

template <int STAGE>
FVK_HD RaggedKeys ragged_keys(const fvk_ragged_args& a, const RaggedReq& q, int i0, int i1) {
    RaggedKeys k;
    const int p0 = a.causal ? q.len - q.nq + i0 : q.len - 1, p1 = a.causal ? q.len - q.nq + i1 : q.len - 1;
    k.hi = p1 + 1 > 0 ? p1 + 1 : 0;
    k.lo = 0;
    k.sink_end = 0;
    k.full_lo = 0;
    k.full_hi = p0 + 1 > 0 ? p0 + 1 : 0;
    if (a.window > 0) {
        const int lo = p0 - a.window + 1, last = p1 - a.window + 1;
        k.lo = lo > 0 ? lo : 0;
        k.full_lo = last > 0 ? last : 0;
        if (a.sink >= k.lo) k.lo = 0;  // one run of keys
        else k.sink_end = a.sink;
        if (a.sink >= k.full_lo) k.full_lo = 0;
    }
    k.lo16 = k.lo & ~15;
    k.n_sink = (k.sink_end + STAGE - 1) / STAGE;
    k.n = k.n_sink + (k.hi > k.lo16 ? (k.hi - k.lo16 + STAGE - 1) / STAGE : 0);
    return k;
}

// first key of stage s; the end of the part of the keys that it belongs to
template <int STAGE>
FVK_HD int ragged_stage(const RaggedKeys& k, int s) { return s < k.n_sink ? s * STAGE : k.lo16 + (s - k.n_sink) * STAGE; }
FVK_HD int ragged_end(const RaggedKeys& k, int s) { return s < k.n_sink ? k.sink_end : k.hi; }

// Block kernel: 16-key group i (0..7) of stage st, a walk that ends in front of stage `end`.  off: its first row from the head's base, in 16-byte units;
// rec: bytes that may be read from there (0: none, the rows arrive as zeros).  It ends with the last key that any row sees, and a page outside the pool has none.
struct RaggedGroup {
    int off, rec;
};
struct RaggedGroups {
    int width, shift, n_pages, end;  // end: one past the last stage of this workgroup
    unsigned ps16, rs16, rs2;        // page and row stride in 16-byte units, row stride in bytes
    unsigned base16;                 // packed keys: the request's first row

    FVK_HD void init(const fvk_ragged_args& a, const RaggedReq& q, int st1, bool paged) {
        width = a.table_width;
        shift = paged ? a.page_shift : 0;
        n_pages = a.n_pages;
        end = st1;
        ps16 = (unsigned)(a.k_ps >> 3);
        rs16 = (unsigned)(a.k_rs >> 3);
        rs2 = (unsigned)(2 * a.k_rs);
        base16 = (unsigned)q.k0 * rs16;
    }
    template <int STAGE>
    FVK_HD int key(const RaggedKeys& ks, int st, int i) const { return ragged_stage<STAGE>(ks, st) + 16 * i; }
    FVK_HD bool in_table(int st, int key) const { return st < end && (key >> shift) < width; }
    template <bool PAGED>
    FVK_HD RaggedGroup at(const RaggedKeys& ks, int st, int key, int page) const {
        const int left = ragged_end(ks, st) - key, rows = left < 16 ? left : 16;
        const bool ok = st < end && left > 0 && (!PAGED || (page >= 0 && page < n_pages));
        const int off = PAGED ? (int)((unsigned)page * ps16 + (unsigned)(key & ((1 << shift) - 1)) * rs16) : (int)(base16 + (unsigned)key * rs16);
        return {ok ? off : 0, ok ? (int)((rows - 1) * rs2 + 256) : 0};
    }
};

// Block kernel: what workgroup `block` takes.  Workgroup x lands on XCD x % 8 (its own L2).  Heads go in teams of four key heads; within every eight ranks
// (places in the order of the batch's blocks) the pairs (head, place in the eight) are dealt to the XCDs in runs of H, team by team.  So an XCD works on a
// few heads, whose blocks read the same pages, but on four key heads rather than one: rows of one head lie Hkv * 256 bytes apart and touch only some of the
// L2's channels.  No gaps: a workgroup without work in front of others leaves a compute unit empty (the dispatcher deals in fixed turns: 228 blocks of
// equal length took two rounds of 256 with gaps).
struct RaggedDeal {
    int run, h, rank;  // run of the key axis, head, place in the order of the blocks; rank < 0: nothing
};
FVK_HD RaggedDeal ragged_deal(const fvk_ragged_args& a, int total, int parts, int block) {
    const int xcd = block & 7, full = total >> 3, G4 = 4 * (a.H / a.Hkv);
    // tasks of an XCD: for every run of the key axis the pairs of the whole eights, then its share of all runs' pairs of the last, incomplete eight
    const int rem = total & 7, whole = full * a.H, left_over = a.H * rem, local = block >> 3;
    int run, row = full, wide = rem, pair;
    if (local < whole * parts) {
        run = parts > 1 ? local / whole : 0;
        pair = local - run * whole;
        row = pair / a.H;
        wide = 8;
        pair += ((row & 1 ? 7 - xcd : xcd) - row) * a.H;  // back and forth: ranks descend in cost
    } else {
        pair = (int)((long)xcd * left_over * parts >> 3) + local - whole * parts;
        if (pair >= (int)((long)(xcd + 1) * left_over * parts >> 3)) return {0, 0, -1};  // the host's bound on the number of blocks is not tight
        run = parts > 1 ? pair / left_over : 0;
        pair -= run * left_over;
    }
    // pair number, team-major: (team, place, member)
    const int team = pair / (wide * G4), members = a.H - team * G4 < G4 ? a.H - team * G4 : G4;
    pair -= team * wide * G4;
    const int place = pair / members;
    return {run, team * G4 + pair - place * members, row * 8 + place};
}
// workgroups for at most n_blocks blocks
FVK_HD unsigned ragged_grid(int H, int n_blocks, int parts) { return 8u * (H * (n_blocks / 8) * parts + (H * (n_blocks % 8) * parts + 7) / 8); }

// Longest walks first (up to 64 requests): blocks in descending order of their cost (stages, an estimate), ties by request.  A request's blocks cost
// min(base + 2 b, cap), b = 0 .. blocks - 1 (a causal block of 256 rows sees two stages more than the one before), or cap each.
struct RaggedCost {
    int causal, blocks, base, cap;
    template <int STAGE>
    FVK_HD void init(const fvk_ragged_args& a, const RaggedReq& q) {
        causal = a.causal;
        blocks = (q.nq + RAGGED_BLOCK - 1) / RAGGED_BLOCK;
        base = cap = 0;
        if (blocks > 0) {
            const int most = a.window > 0 ? (int)(((unsigned)a.window + (unsigned)a.sink + (a.causal ? 2 * STAGE : STAGE)) / STAGE) : 0x10000000;
            cap = (q.len + STAGE - 1) / STAGE;
            base = a.causal ? cap - 2 * (blocks - 1) : cap;
            cap = cap < most ? cap : most;
        }
    }
    FVK_HD int least() const { return blocks > 0 ? (base < cap ? base : cap) : 0x10000000; }
    FVK_HD int most() const { return blocks > 0 ? cap : -0x10000000; }
    FVK_HD int at_least(int t) const {  // blocks that cost t or more: the last ones
        const int skip = causal ? (t - base + 1) >> 1 : t > base ? blocks : 0;
        const int n = blocks - (skip > 0 ? skip : 0);
        return t > cap || n < 0 ? 0 : n;
    }
};

// Rows kernel: 16-key half group from `key` on, seen up to kmax.  Offsets of its first row (elements) and the bytes from there that a descriptor covers; a
// page outside the pool, or a key behind the last one, has none.  Rows outside [kmin, kmax) are left out by the lanes themselves.
struct RaggedHalf {
    long k, v;
    unsigned k_rec, v_rec;
};
template <bool PAGED>
FVK_HD RaggedHalf ragged_half(const fvk_ragged_args& a, int key, int kmax, int page) {
    RaggedHalf h;
    const int in_page = PAGED ? key & ((1 << a.page_shift) - 1) : key;
    const bool in = PAGED ? page >= 0 && page < a.n_pages : key < kmax;
    h.k = in ? (PAGED ? (long)page * a.k_ps : 0) + (long)in_page * a.k_rs : 0;
    h.v = in ? (PAGED ? (long)page * a.v_ps : 0) + (long)in_page * a.v_rs : 0;
    h.k_rec = in ? 15 * (unsigned)(a.k_rs * 2) + 256 : 0;
    h.v_rec = in ? 15 * (unsigned)(a.v_rs * 2) + 256 : 0;
    return h;
}

}  // namespace fvk
