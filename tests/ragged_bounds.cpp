// The ragged attention kernels' whole-number arithmetic (fastvideo_amd/csrc/ragged_walk.h) on the CPU, over random lengths, windows, sinks, strides, page
// sizes and wrong metadata: every row, table entry and key address that the kernels form lies inside its tensor, every key that a row sees is read from its
// own place, and every (head, block of rows, run of keys) of a batch with right metadata is taken by exactly one workgroup.
// usage: ragged_bounds SEED CASES
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../fastvideo_amd/csrc/ragged_walk.h"

using namespace fvk;

static std::mt19937_64 rng;
static long pick(long lo, long hi) { return lo + (long)(rng() % (unsigned long)(hi - lo + 1)); }
static long wide(long lo, long hi) { return pick(0, 2) ? pick(lo, std::min(hi, lo + 40)) : pick(lo, hi); }

#define HOLDS(x)                                                                                                                                        \
    do {                                                                                                                                                \
        if (!(x)) {                                                                                                                                     \
            printf("line %d: %s\n  T=%d R=%d H=%d Hkv=%d table_width=%d page_shift=%d n_pages=%d total_k=%d causal=%d window=%d sink=%d k_ps=%ld "        \
                   "k_rs=%ld k_hs=%ld v_ps=%ld v_rs=%ld v_hs=%ld\n",                                                                                       \
                   __LINE__, #x, a.T, a.R, a.H, a.Hkv, a.table_width, a.page_shift, a.n_pages, a.total_k, a.causal, a.window, a.sink, a.k_ps, a.k_rs,      \
                   a.k_hs, a.v_ps, a.v_rs, a.v_hs);                                                                                                       \
            exit(1);                                                                                                                                     \
        }                                                                                                                                                \
    } while (0)

static long n_pieces, n_halves, n_deals;  // what was looked at

constexpr int KT = 128, ST = 32;  // keys per stage: block kernel, rows kernel

struct Extent {  // bytes of K (or V) behind the tensor's first element
    long ps, rs, hs;
    long bytes(const fvk_ragged_args& a) const {
        const bool paged = a.block_table != nullptr;
        const long rows = paged ? 1L << a.page_shift : a.total_k, pages = paged ? a.n_pages : 1;
        return pages > 0 && rows > 0 ? 2 * ((pages - 1) * ps + (rows - 1) * rs + (a.Hkv - 1) * hs + 128) : 0;
    }
};
// where key `key` of a request lies, or -1
static long place(const fvk_ragged_args& a, const Extent& e, const RaggedReq& q, int r, int key) {
    if (!a.block_table) return 2 * (long)(q.k0 + key) * e.rs;
    const int page = a.block_table[(long)r * a.table_width + (key >> a.page_shift)];
    return page < 0 || page >= a.n_pages ? -1 : 2 * ((long)page * e.ps + (long)(key & ((1 << a.page_shift) - 1)) * e.rs);
}

template <bool PAGED>
static void block_kernel(const fvk_ragged_args& a, int parts, bool right, int samples) {
    const Extent K{a.k_ps, a.k_rs, a.k_hs};
    const long room = K.bytes(a), n_blocks_l = (a.T + 255L) / 256 + a.R - 1;
    if ((n_blocks_l + 8) * a.H * parts > 0x7fffffL) return;  // the host takes the rows kernel
    const long reach = PAGED ? (a.n_pages > 0 ? a.n_pages - 1L : 0L) * a.k_ps + 256L * a.k_rs : (a.total_k + 1024L) * a.k_rs;
    if (reach / 8 > 0xffffffffL) return;
    const int n_blocks = (int)n_blocks_l, G = a.H / a.Hkv;
    std::vector<RaggedReq> req(a.R);
    std::vector<RaggedCost> cost(a.R);
    unsigned sum = 0;  // (wraps as the kernel's does)
    long real = 0;
    for (int r = 0; r < a.R; ++r) {
        req[r] = ragged_req<PAGED>(a, r);
        HOLDS(req[r].q0 >= 0 && req[r].nq >= 0 && req[r].q0 + req[r].nq <= a.T);
        cost[r].init<KT>(a, req[r]);
        sum += cost[r].blocks;
        real += cost[r].blocks;
    }
    const int total = (int)sum;
    if (right) HOLDS(total <= n_blocks);
    const unsigned grid = ragged_grid(a.H, n_blocks, parts);
    const bool all = right && grid <= 4096;
    std::vector<int> taken(all ? (size_t)total * a.H * parts : 0);
    std::vector<char> seen_block(all ? (size_t)a.R * (n_blocks + 1) : 0);
    for (unsigned s = 0; s < (all ? grid : (unsigned)samples); ++s) {
        const unsigned block = all ? s : (unsigned)pick(0, grid - 1);
        const RaggedDeal d = ragged_deal(a, total, parts, (int)block);
        if (d.rank < 0) continue;
        ++n_deals;
        HOLDS(d.h >= 0 && d.h < a.H && d.run >= 0 && d.run < parts && d.rank < real);
        if (right) HOLDS(d.rank < total);
        if (all) HOLDS(++taken[((size_t)d.run * a.H + d.h) * total + d.rank] == 1);
        int r = -1, index = 0, rank = d.rank;
        if (a.R <= 64) {
            HOLDS(d.rank < total);
            int lo = 0x10000000, hi = -0x10000000;
            for (int i = 0; i < a.R; ++i) lo = std::min(lo, cost[i].least()), hi = std::max(hi, cost[i].most());
            ++hi;
            auto count = [&](int t) {
                int n = 0;
                for (int i = 0; i < a.R; ++i) n += cost[i].at_least(t);
                return n;
            };
            while (hi - lo > 1) {
                const int mid = lo + ((hi - lo) >> 1);
                if (count(mid) > rank) lo = mid;
                else hi = mid;
            }
            rank -= count(lo + 1);
            HOLDS(rank >= 0);
            int upto = 0;
            for (int i = 0; i < a.R && r < 0; ++i) {
                const int above = cost[i].at_least(lo + 1), same = cost[i].at_least(lo) - above;
                upto += same;
                if (upto > rank) r = i, index = cost[i].blocks - 1 - above - (rank - (upto - same));
            }
            HOLDS(r >= 0);
        } else {
            for (int i = 0; i < a.R && r < 0; ++i) {
                if (cost[i].blocks > rank) r = i, index = rank;
                else rank -= cost[i].blocks;
            }
            if (r < 0) continue;
        }
        HOLDS(index >= 0 && index < cost[r].blocks);
        if (all && d.h == 0 && d.run == 0) {
            char& c = seen_block[(size_t)r * (n_blocks + 1) + index];
            HOLDS(c == 0);
            c = 1;
        }
        const RaggedReq q = req[r];
        const int first_row = index * 256, last_row = first_row + 256 < q.nq ? first_row + 255 : q.nq - 1;
        HOLDS(first_row <= last_row && q.q0 + last_row < a.T);
        const RaggedKeys ks = ragged_keys<KT>(a, q, first_row, last_row);
        const int st0 = (int)((long)ks.n * d.run / parts), st1 = (int)((long)ks.n * (d.run + 1) / parts), n = st1 - st0;
        HOLDS(ks.n >= 0 && ks.hi <= q.len && ks.sink_end <= ks.lo && ks.lo >= 0 && (ks.n == 0 || ks.lo16 <= ks.hi));
        if (n <= 0) continue;
        RaggedGroups g;
        g.init(a, q, st1, PAGED);
        const long base = 2L * (d.h / G) * a.k_hs;
        // the prologue issues stages 0 and 1, pair j issues stage j + 2 of K and j + 1 of V; the next eight stages' page ids are loaded eight stages ahead
        for (int st = 0; st <= n + 8; ++st) {
            if (n > 40 && st > 20 && st < n - 12 && !(st % 7 == 0)) continue;
            for (int i = 0; i < 8; ++i) {
                const int s_ = st0 + st, key = g.key<KT>(ks, s_, i);
                int page = -1;
                if (PAGED && g.in_table(s_, key)) {
                    HOLDS(key >= 0 && (key >> a.page_shift) < a.table_width);
                    page = a.block_table[(long)r * a.table_width + (key >> a.page_shift)];
                }
                const RaggedGroup at = g.at<PAGED>(ks, s_, key, PAGED ? page : 0);
                if (st >= n) HOLDS(at.rec == 0);
                if (at.rec == 0) continue;
                ++n_pieces;
                HOLDS(at.rec > 0 && (unsigned)at.rec < 0x80000000u);
                const long from = base + 16L * (unsigned)at.off;
                HOLDS(from >= 0 && from + at.rec <= room);
                // every lane's 16 bytes, of K and V: inside the group's records or not read at all; a key that a row sees comes from its own place
                const int end = ragged_end(ks, s_);
                for (int row = 0; row < 16; ++row) {
                    const unsigned rs2 = (unsigned)(2 * a.k_rs), far = (unsigned)row * rs2 + 240;
                    if (key + row < end) {
                        HOLDS(far + 16 <= (unsigned)at.rec);
                        HOLDS(from + (long)row * rs2 == base + place(a, K, q, r, key + row));
                    } else if (rs2 >= 256) {
                        HOLDS((unsigned)row * rs2 + 16 > (unsigned)at.rec);  // behind the last key: zeros
                    }
                }
            }
        }
    }
    if (all) {
        for (int c : taken) HOLDS(c == 1);
        if (total > 0)
            for (int r = 0; r < a.R; ++r)
                for (int b = 0; b < cost[r].blocks; ++b) HOLDS(seen_block[(size_t)r * (n_blocks + 1) + b] == 1);
    }
}

template <bool PAGED>
static void rows_kernel(const fvk_ragged_args& a, int qb, int parts, bool right, int samples) {
    const Extent K{a.k_ps, a.k_rs, a.k_hs}, V{a.v_ps, a.v_rs, a.v_hs};
    const long k_room = K.bytes(a), v_room = V.bytes(a);
    const int G = a.H / a.Hkv, tile = 16 * qb;
    long tiles = 0;
    for (int r = 0; r < a.R; ++r) tiles += ((long)ragged_req<PAGED>(a, r).nq * G + tile - 1) / tile;
    if (right) HOLDS(tiles <= (long)a.T * G / tile + a.R);  // the host's bound, where gridDim.z counts tiles
    for (int s = 0; s < samples; ++s) {
        const int r = (int)pick(0, a.R - 1), kvh = (int)pick(0, a.Hkv - 1), part = (int)pick(0, parts - 1);
        const RaggedReq q = ragged_req<PAGED>(a, r);
        const long rows_l = (long)q.nq * G;
        if (rows_l == 0 || rows_l > 0x7fffffffL) continue;
        const int rows = (int)rows_l, rb = (int)pick(0, (rows - 1) / tile), row0 = rb * tile, row1 = std::min(row0 + tile, rows);
        HOLDS(q.q0 + (row1 - 1) / G < a.T);
        const RaggedKeys ks = ragged_keys<ST>(a, q, row0 / G, (row1 - 1) / G);
        const int st0 = (int)((long)ks.n * part / parts), st1 = (int)((long)ks.n * (part + 1) / parts);
        for (int st = st0; st < st1; ++st) {
            if (st - st0 > 12 && st1 - st > 6) continue;
            for (int half = 0; half < 2; ++half) {
                const int key = ragged_stage<ST>(ks, st) + 16 * half, kmin = st < ks.n_sink ? 0 : ks.lo, kmax = ragged_end(ks, st);
                int page = 0;
                if (PAGED) {
                    page = -1;
                    if (key < kmax) {
                        HOLDS(key >= 0 && (key >> a.page_shift) < a.table_width);
                        page = a.block_table[(long)r * a.table_width + (key >> a.page_shift)];
                    }
                }
                const RaggedHalf h = ragged_half<PAGED>(a, key, kmax, page);
                const long kb = 2 * ((long)kvh * a.k_hs + (PAGED ? 0 : (long)q.k0 * a.k_rs)), vb = 2 * ((long)kvh * a.v_hs + (PAGED ? 0 : (long)q.k0 * a.v_rs));
                ++n_halves;
                HOLDS(h.k_rec < 0x80000000u && h.v_rec < 0x80000000u);
                for (int row = 0; row < 16; ++row) {
                    if (key + row < kmin || key + row >= kmax || h.k_rec == 0) continue;  // the lane's offset passes every descriptor, or there are no records
                    const unsigned kf = (unsigned)(row * a.k_rs * 2) + 240, vf = (unsigned)(row * a.v_rs * 2) + 240;
                    HOLDS(kf + 16 <= h.k_rec && vf + 16 <= h.v_rec);
                    const long kp = kb + 2 * h.k + (long)row * a.k_rs * 2, vp = vb + 2 * h.v + (long)row * a.v_rs * 2;
                    HOLDS(kp >= 0 && kp + 256 <= k_room && vp >= 0 && vp + 256 <= v_room);
                    HOLDS(kp == 2L * kvh * a.k_hs + place(a, K, q, r, key + row) && vp == 2L * kvh * a.v_hs + place(a, V, q, r, key + row));
                }
            }
        }
    }
}

static void one_case(int c) {
    fvk_ragged_args a{};
    const bool paged = pick(0, 2) != 0, right = pick(0, 3) != 0, huge = pick(0, 19) == 0;
    a.Hkv = (int)(pick(0, 3) ? pick(1, 8) : pick(1, 40));
    a.H = a.Hkv * (int)pick(1, 5);
    a.R = (int)(pick(0, 3) ? pick(1, 9) : pick(1, huge ? 4000 : 150));
    a.causal = paged && pick(0, 1);
    std::vector<int32_t> cu(a.R + 1), len(paged ? a.R : a.R + 1), table;
    long T = 0;
    for (int r = 0; r < a.R; ++r) {
        cu[r] = (int)T;
        T += pick(0, 4) == 0 ? 0 : pick(0, 2) ? pick(1, 70) : pick(1, a.R > 100 ? 600 : 3000);
    }
    cu[a.R] = (int)T;
    if (huge) T += 100000000;
    a.T = (int)(T + pick(0, 5));
    if (a.T == 0) a.T = 1;
    if (paged) {
        a.page_shift = (int)pick(4, 8);
        a.table_width = (int)(pick(0, 3) ? pick(1, 60) : pick(1, a.R > 100 ? 300 : 3000));
        a.n_pages = (int)(huge ? pick(1, 1 << 22) : wide(0, 5000));
        table.resize((size_t)a.R * a.table_width);
        for (auto& t : table) t = a.n_pages && pick(0, 9) ? (int)pick(0, a.n_pages - 1) : (int)pick(-2, 1) * (int)pick(1, 0x7fffffff / 2);
        for (auto& l : len) l = (int)(pick(0, 5) == 0 ? 0 : wide(0, (long)a.table_width << a.page_shift));
    } else {
        long S = 0;
        for (int r = 0; r < a.R; ++r) {
            len[r] = (int)S;
            S += pick(0, 4) == 0 ? 0 : pick(0, 2) ? pick(1, 150) : pick(1, 4000);
        }
        len[a.R] = (int)S;
        a.total_k = (int)(S + pick(0, 3));
    }
    // strides: page-row-head, head-row, a fused projection's views, rows that overlap
    const long page = paged ? 1L << a.page_shift : a.total_k;
    const int layout = (int)pick(0, 3);
    a.k_rs = layout == 1 ? 128 : layout == 3 ? 8 * pick(0, 40) : (a.Hkv + (layout == 2 ? 8 * pick(0, 5) : 0)) * 128L;
    a.k_hs = layout == 1 ? page * 128 : 128;
    a.k_ps = paged ? (layout == 1 ? page * 128 * a.Hkv : page * a.k_rs + 8 * pick(0, 3)) : 0;
    a.v_ps = a.k_ps, a.v_rs = a.k_rs, a.v_hs = a.k_hs;
    const bool same = pick(0, 3) != 0;
    if (!same) a.v_rs += 128, a.v_ps += page * 128 + 8;
    if (huge && pick(0, 1)) a.k_rs = a.v_rs = 1 << 24, a.k_ps = a.v_ps = paged ? page << 24 : 0;
    if (paged && pick(0, 1)) {
        a.window = (int)(pick(0, 5) ? wide(1, 3000) : pick(0, 1) ? 0x3fffffff : pick(1, 0x3fffffff));
        a.sink = (int)(pick(0, 2) ? 0 : pick(0, 5) ? wide(0, 2000) : 0x3fffffff);
    }
    if (!right) {  // anything
        for (auto* v : {&cu, &len})
            for (auto& x : *v)
                if (pick(0, 2) == 0) x = (int)(pick(0, 1) ? pick(-0x7fffffffL - 1, 0x7fffffff) : pick(-5, a.T + 5));
    }
    a.cu_q = cu.data();
    a.kv_lens = len.data();
    a.block_table = paged ? table.data() : nullptr;
    a.max_q = a.max_kv = 1;
    const int parts = (int)(pick(0, 1) ? 1 : pick(2, 16)), samples = 24;
    if (same) paged ? block_kernel<true>(a, parts, right, samples) : block_kernel<false>(a, parts, right, samples);
    for (int qb = 1; qb <= 4; qb *= 2) paged ? rows_kernel<true>(a, qb, (int)pick(1, 64), right, samples) : rows_kernel<false>(a, qb, (int)pick(1, 64), right, samples);
    (void)c;
}

// total blocks that pass 2^31: overlapping requests of a batch at the size limit
static void overlapping() {
    std::vector<int32_t> cu(65536), len(65535, 100), table(65535, 0);
    for (int r = 0; r < 65536; ++r) cu[r] = r & 1 ? 0x3fffffff : 0;
    fvk_ragged_args a{};
    a.T = 0x3fffffff, a.R = 65535, a.H = a.Hkv = 1, a.table_width = 1, a.page_shift = 4, a.n_pages = 1, a.k_rs = a.v_rs = 128, a.k_ps = a.v_ps = 2048, a.k_hs = a.v_hs = 128;
    a.cu_q = cu.data(), a.kv_lens = len.data(), a.block_table = table.data();
    block_kernel<true>(a, 1, false, 2000);
    a.R = 64;
    block_kernel<true>(a, 1, false, 2000);
}

int main(int argc, char** argv) {
    const int seed = argc > 1 ? atoi(argv[1]) : 0, cases = argc > 2 ? atoi(argv[2]) : 1000;
    rng.seed(seed);
    for (int c = 0; c < cases; ++c) one_case(c);
    overlapping();
    printf("%d cases hold: %ld workgroups, %ld pieces of 16 keys, %ld halves of the rows kernel\n", cases, n_deals, n_pieces, n_halves);
}
