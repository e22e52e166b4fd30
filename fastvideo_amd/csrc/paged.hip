// The paged cache's own passes: the page plan of a step (block tables, slot map, positions) and the fused QK-norm + three-axis RoPE pass that writes
// the new keys and values into their pages.  The attention that reads the pages: attn_rows.hip, attn_ragged.hip.
#include "fvk_common.h"

namespace {

// ------------------------------------------------------------------ plan
// All whole numbers.  With new = the request's tokens that the batch holds (those beyond n_tokens are dropped: they have no row, so no key and no page),
// total = start + new, pages = ceil(total / P), need = max(0, pages - held):
//   a request is GRANTED iff its pages fit the table's width and (need = 0 or (sum of the needs before it) + need <= free_count);
//   its i-th new page is free[count - 1 - off - i];  a page is dead once no row of this step or a later one can see it (window, sink) and goes back
//   onto the stack in (request, page) order.
// Bound: a few KB to a few MB, so launch latency; hence ONE launch for everything that does not depend on the number of dead pages (every workgroup
// repeats the prefix sums over the requests: 2 loads and 8 shuffles for up to 256 of them, cheaper than a second launch), and a second one only when there
// is a window.  Measured: 4.2 us for 4 streams of one token, 6.2 + 4.2 us for 48 rollouts of 145 000 tokens with a window (1000 cells a row).
struct PlanArgs {
    const int32_t *starts, *new_lens, *table, *held, *free_in, *count;
    int32_t *table_out, *held_out, *free_out, *count_out, *cu_q, *kv_lens, *slots, *positions, *granted;
    int32_t* scratch;  // dead pages per request [R], needs before it [R], the stack's height without the taken pages; nullptr: no window
    int R, width, n_free, page, n_tokens, gh, gw, window, sink, causal;
    int table_blocks;  // workgroups that copy table rows; the others handle tokens and the stack
    int row_waves;     // waves of a workgroup that share a table row: 1 or 4 (a wide table: 16 loads of one wave, one after the other, otherwise)
};

constexpr int PLAN_MAX_R = 4096;

struct PlanReq {
    long total;
    int start, add, pages, need, held, fits;
};

// add: rows of the batch that the request has, cu[r + 1] - cu[r]
__device__ __forceinline__ PlanReq plan_req(const PlanArgs& a, int r, int add) {
    PlanReq q;
    const int s = a.starts[r], h = a.held[r];
    q.start = s > 0 ? s : 0;
    q.add = add;
    q.held = h > 0 ? h : 0;
    q.total = (long)q.start + q.add;
    const long pages = (q.total + a.page - 1) / a.page;
    q.fits = pages <= a.width;
    q.pages = q.fits ? (int)pages : 0;
    q.need = q.pages > q.held ? q.pages - q.held : 0;
    return q;
}

// dead pages of a granted request are the j in [first, last): j * P >= sink and (j + 1) * P <= low
__device__ __forceinline__ void plan_dead_range(const PlanArgs& a, const PlanReq& q, int& first, int& last) {
    first = last = 0;
    if (a.window <= 0) return;
    const long low = q.total - a.window + (a.causal ? 1 - q.add : 0);
    if (low <= 0) return;
    first = (int)(((long)a.sink + a.page - 1) / a.page);
    const long l = low / a.page;
    last = l < a.width ? (int)l : a.width;
}

__device__ __forceinline__ int plan_page(const PlanArgs& a, const PlanReq& q, int r, int off, bool granted, int count, int j) {
    if (granted && j >= q.held && j < q.pages) {
        const int at = count - 1 - (off + j - q.held);
        return at >= 0 && at < a.n_free ? a.free_in[at] : -1;
    }
    return a.table[(long)r * a.width + j];
}

// Exclusive prefix sums over the requests by the whole workgroup (256 threads): new tokens, clamped to n_tokens, into cu[0..R], and the pages that the
// tokens within the batch need into off[0..R].  Both in one pass, which is right where the batch holds all tokens; where it does not, the pages again with
// the tokens that are left (a pass that waits for the tokens' sums first costs 10 % at 4096 requests).
__device__ void plan_scan(const PlanArgs& a, int* cu, int* off) {
    __shared__ long wsum_t[4];
    __shared__ int wsum_p[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    long base_t = 0;
    int base_p = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int r0 = 0; r0 < a.R; r0 += 256) {
            const int r = r0 + tid;
            long t = 0;
            int p = 0;
            if (r < a.R) {
                if (pass == 0) {
                    const int n = a.new_lens[r];
                    t = n > 0 ? n : 0;
                }
                p = plan_req(a, r, pass == 0 ? (int)(t < a.n_tokens ? t : a.n_tokens) : cu[r + 1] - cu[r]).need;
            }
            const long t0 = t;
            const int p0 = p;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const long tu = __shfl_up(t, o, 64);
                const int pu = __shfl_up(p, o, 64);
                if (lane >= o) { t += tu; p += pu; }
            }
            if (lane == 63) { wsum_t[wave] = t; wsum_p[wave] = p; }
            __syncthreads();
            long bt = base_t;
            int bp = base_p;
            for (int w = 0; w < 4; ++w) {
                if (w < wave) { bt += wsum_t[w]; bp += wsum_p[w]; }
                base_t += wsum_t[w];
                base_p += wsum_p[w];
            }
            if (r < a.R) {
                const long c = bt + t - t0;
                if (pass == 0) cu[r] = (int)(c < a.n_tokens ? c : a.n_tokens);
                off[r] = bp + p - p0;
            }
            __syncthreads();
        }
        if (tid == 0) {
            if (pass == 0) cu[a.R] = (int)(base_t < a.n_tokens ? base_t : a.n_tokens);
            off[a.R] = base_p;
        }
        __syncthreads();
        if (base_t <= a.n_tokens) return;  // (the same in all threads)
        base_p = 0;
    }
}

__device__ __forceinline__ bool plan_granted(const PlanReq& q, int off, int count) { return q.fits && (q.need == 0 || (long)off + q.need <= count); }

__device__ __forceinline__ int plan_count(const PlanArgs& a) {
    const int c = a.count[0];
    return c < 0 ? 0 : (c < a.n_free ? c : a.n_free);
}

// pages taken off the stack: the granted needs form a prefix of the requests (the first refusal of a need refuses every later one)
__device__ int plan_taken(const PlanArgs& a, const int* cu, const int* off, int count) {
    int lo = 0;
    for (int r = threadIdx.x; r < a.R; r += 256) {
        const PlanReq q = plan_req(a, r, cu[r + 1] - cu[r]);
        if (q.need > 0 && plan_granted(q, off[r], count) && off[r] + q.need > lo) lo = off[r] + q.need;
    }
    __shared__ int best[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int v = __shfl_xor(lo, o, 64);
        lo = v > lo ? v : lo;
    }
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = lo;
    __syncthreads();
    lo = best[0];
    for (int w = 1; w < 4; ++w) lo = best[w] > lo ? best[w] : lo;
    __syncthreads();
    return lo;
}

__global__ __launch_bounds__(256) void paged_plan_kernel(PlanArgs a) {
    __shared__ int cu[PLAN_MAX_R + 1], off[PLAN_MAX_R + 1];
    plan_scan(a, cu, off);
    const int tid = threadIdx.x;
    const int count = plan_count(a);
    if ((int)blockIdx.x < a.table_blocks) {  // one wave or one workgroup per request: its table row
        const bool shared = a.row_waves > 1;
        const int r = shared ? blockIdx.x : blockIdx.x * 4 + (tid >> 6), lane = shared ? tid : tid & 63, step = shared ? 256 : 64;
        if (r >= a.R) return;  // (a shared row's workgroup has one request: all of it leaves)
        const PlanReq q = plan_req(a, r, cu[r + 1] - cu[r]);
        const bool ok = plan_granted(q, off[r], count);
        int first, last, dead = 0;
        plan_dead_range(a, q, first, last);
#pragma unroll 4
        for (int j = lane; j < a.width; j += step) {
            int p = plan_page(a, q, r, off[r], ok, count, j);
            if (ok && j >= first && j < last && p >= 0) {
                ++dead;
                p = -1;
            }
            a.table_out[(long)r * a.width + j] = p;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) dead += __shfl_xor(dead, o, 64);
        if (shared) {
            __shared__ int sums[4];
            if ((tid & 63) == 0) sums[tid >> 6] = dead;
            __syncthreads();
            dead = sums[0] + sums[1] + sums[2] + sums[3];
        }
        if (lane == 0) {
            a.held_out[r] = ok && q.pages > q.held ? q.pages : a.held[r];
            a.kv_lens[r] = ok ? (int)q.total : 0;
            a.granted[r] = ok;
            a.cu_q[r + 1] = cu[r + 1];
            if (r == 0) a.cu_q[0] = 0;
            if (a.scratch) {
                a.scratch[r] = dead;
                a.scratch[a.R + r] = off[r];
            }
        }
        return;
    }
    const int block = blockIdx.x - a.table_blocks, blocks = gridDim.x - a.table_blocks;
    if (block == 0) {
        const int taken = plan_taken(a, cu, off, count);
        if (tid == 0) {
            a.count_out[0] = count - taken;  // the second launch adds the dead pages
            if (a.scratch) a.scratch[2 * a.R] = count - taken;
        }
    }
    for (long i = block * 256L + tid; i < a.n_free; i += blocks * 256L) a.free_out[i] = a.free_in[i];
    const int frame = a.gh * a.gw;
    for (long i = block * 256L + tid; i < a.n_tokens; i += blocks * 256L) {
        int slot = -1, pos = 0;
        if (i < cu[a.R]) {
            int lo = 0, hi = a.R;  // the request r with cu[r] <= i < cu[r + 1]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= i) lo = mid;
                else hi = mid;
            }
            const PlanReq q = plan_req(a, lo, cu[lo + 1] - cu[lo]);
            const long at = (long)q.start + (i - cu[lo]);
            pos = (int)(at < 0x7fffffffL ? at : 0x7fffffffL);
            if (plan_granted(q, off[lo], count)) {
                const int j = pos / a.page;
                int first, last;
                plan_dead_range(a, q, first, last);
                const int p = j >= first && j < last ? -1 : plan_page(a, q, lo, off[lo], true, count, j);
                if (p >= 0) slot = p * a.page + (pos - j * a.page);
            }
        }
        a.slots[i] = slot;
        const int f = pos / frame, rest = pos - f * frame, y = rest / a.gw;
        a.positions[i * 3] = f;
        a.positions[i * 3 + 1] = y;
        a.positions[i * 3 + 2] = rest - y * a.gw;
    }
}

// the dead pages go back onto the stack: one wave per request, its place from the prefix sum of the counts.  What the first launch knows comes from the
// scratch (a second prefix sum over the requests cost 1.3 of 5.3 us).
__global__ __launch_bounds__(256) void paged_release_kernel(PlanArgs a) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int r = blockIdx.x * 4 + (tid >> 6);
    if (r >= a.R) return;
    const int count = plan_count(a), left = a.scratch[2 * a.R], off = a.scratch[a.R + r];
    int before = 0, all = 0;
    for (int i = lane; i < a.R; i += 64) {
        const int c = a.scratch[i];
        all += c;
        before += i < r ? c : 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        before += __shfl_xor(before, o, 64);
        all += __shfl_xor(all, o, 64);
    }
    if (r == 0 && lane == 0) a.count_out[0] = left + all < a.n_free ? left + all : a.n_free;
    const PlanReq q = plan_req(a, r, a.cu_q[r + 1] - a.cu_q[r]);  // (of the first launch)
    int first, last, at = left + before;
    plan_dead_range(a, q, first, last);
    if (a.scratch[r] == 0) return;  // nothing dead, or not granted
    for (int j0 = first; j0 < last; j0 += 256) {  // four loads in flight
        int p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + 64 * i + lane;
            p[i] = j < last ? plan_page(a, q, r, off, true, count, j) : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned long long live = __ballot(p[i] >= 0);
            const int to = at + __popcll(live & ((1ull << lane) - 1));
            if (p[i] >= 0 && to >= 0 && to < a.n_free) a.free_out[to] = p[i];
            at += __popcll(live);
        }
    }
}

// ------------------------------------------------------------------ norm + rotary + page write
// y = x * rsqrt(mean(x^2) + eps) * w over the whole row, then every pair (a, b) of a head's columns turned by the angle of its axis at the token's own
// (t, h, w):  (a cos - b sin, b cos + a sin).  HBM-bound: every q, k, v element is read once and written once (86 MB for a block of three 480p frames of
// 12 heads).  One wave per (token, tensor): the row stays in registers between the sum of squares and the rotation, and a lane's eight columns
// of a head are the same eight in every head (64 lanes x 8 columns = 4 heads per step), so its four (cos, sin) pairs are fetched once per row.
// Rounded once, at the store; round_norm = 1 adds the two roundings of the eager layer (normalised value, weighted value), so that the batched path
// caches the bits that the one-sample path caches.
// Measured: 17.7 us for that block (4.9 TB/s; a large copy reaches 4.8), 152 us for 12 390 tokens of 40 heads (761 MB, 5.0 TB/s), 5.6 us for 16 tokens; with
// round_norm 0.4 .. 1.7 us more.
struct WriteArgs {
    const bf16_t* in[3];
    const bf16_t* w[2];
    const int32_t* positions;
    const float2* rope;
    const int32_t* slots;
    bf16_t *q_out, *k_pages, *v_pages;
    long q_stride, k_stride, v_stride, out_stride;
    long kp_page, kp_row, kp_head, vp_page, vp_row, vp_head;
    int T, H, Hkv, pairs, n0, n1, n2, p0, p1;  // p0, p1: first pair of the second / third axis
    int page_shift, n_pages, round_norm;
    float eps;
};

template <int VPL>
__global__ __launch_bounds__(256) void rmsnorm_rope_paged_kernel(WriteArgs a) {
#pragma clang fp contract(off)  // products and sums rounded one by one, as rmsnorm_rope_kernel computes them: the same bits with round_norm
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.T) return;
    const int t = blockIdx.y;
    const int slot = t > 0 ? a.slots[row] : 0;  // (used below: the row's loads do not wait for it)
    const int heads = t == 0 ? a.H : a.Hkv;
    const int nchunks = heads * 16;
    const bf16_t* in = a.in[t] + (long)row * (t == 0 ? a.q_stride : t == 1 ? a.k_stride : a.v_stride);
    bf16x8 x[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * i;
        if (c < nchunks) x[i] = ld_bf16x8(in + c * 8);
    }
    if (slot < 0 || (slot >> a.page_shift) >= a.n_pages) return;  // a padding row, or no page of the pool
    const long in_page = slot & ((1 << a.page_shift) - 1);
    bf16_t* out = t == 0 ? a.q_out + (long)row * a.out_stride
                         : t == 1 ? a.k_pages + (long)(slot >> a.page_shift) * a.kp_page + in_page * a.kp_row
                                  : a.v_pages + (long)(slot >> a.page_shift) * a.vp_page + in_page * a.vp_row;
    const long head_stride = t == 0 ? 128 : t == 1 ? a.kp_head : a.vp_head;
    if (t == 2) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int c = lane + 64 * i;
            if (c < nchunks) st_bf16x8(out + (c >> 4) * head_stride + (c & 15) * 8, x[i]);
        }
        return;
    }
    float2 turn[4] = {};
    if (a.rope) {
        const int pt = a.positions[row * 3L], ph = a.positions[row * 3L + 1], pw = a.positions[row * 3L + 2];
        const bool known = pt >= 0 && pt < a.n0 && ph >= 0 && ph < a.n1 && pw >= 0 && pw < a.n2;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = (lane & 15) * 4 + j;
            const long r = p < a.p0 ? (long)pt * a.pairs + p : p < a.p1 ? (long)(a.n0 + ph) * a.pairs + p - a.p0 : (long)(a.n0 + a.n1 + pw) * a.pairs + p - a.p1;
            // a position outside the table has no angle: the row comes out as NaN, nothing is read outside the table
            turn[j] = known ? a.rope[r] : make_float2(__builtin_nanf(""), __builtin_nanf(""));
        }
    }
    const bf16_t* w = a.w[t];
    float scale = 1.f;
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (lane + 64 * i < nchunks)
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += (float)x[i][j] * (float)x[i][j];
        scale = rsqrtf(wave_sum(ss) / (float)(heads * 128) + a.eps);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int c = lane + 64 * i;
        if (c >= nchunks) continue;
        float v[8];
        if (w) {
            const bf16x8 wv = ld_bf16x8(w + c * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = (float)x[i][j] * scale;
                v[j] = a.round_norm ? bf16_round(bf16_round(v[j]) * (float)wv[j]) : v[j] * (float)wv[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)x[i][j];
        }
        bf16x8 o;
        if (a.rope) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float2 cs = turn[j >> 1];
                o[j] = (bf16_t)(v[j] * cs.x + (-v[j + 1]) * cs.y);
                o[j + 1] = (bf16_t)(v[j + 1] * cs.x + v[j] * cs.y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = (bf16_t)v[j];
        }
        st_bf16x8(out + (c >> 4) * head_stride + (c & 15) * 8, o);
    }
}

template <typename F>
int dispatch_heads(int chunks, F&& f) {
    const int need = (chunks + 63) / 64;
    if (need <= 1) return f(std::integral_constant<int, 1>{});
    if (need <= 2) return f(std::integral_constant<int, 2>{});
    if (need <= 3) return f(std::integral_constant<int, 3>{});
    if (need <= 4) return f(std::integral_constant<int, 4>{});
    if (need <= 6) return f(std::integral_constant<int, 6>{});
    if (need <= 10) return f(std::integral_constant<int, 10>{});
    if (need <= 16) return f(std::integral_constant<int, 16>{});
    return FVK_ERR_ARG;
}

int page_shift_of(int page) {
    for (int s = 4; s <= 8; ++s)
        if (page == 1 << s) return s;
    return -1;
}

}  // namespace

extern "C" int fvk_paged_plan(const int32_t* starts, const int32_t* new_lens, const int32_t* block_table, const int32_t* pages_held,
                              const int32_t* free_pages, const int32_t* free_count, int32_t* table_out, int32_t* held_out, int32_t* free_out,
                              int32_t* count_out, int32_t* cu_q, int32_t* kv_lens, int32_t* slot_map, int32_t* positions, int32_t* granted,
                              int32_t* dead_counts, int n_requests, int table_width, int n_free, int page_size, int n_tokens, int grid_h, int grid_w,
                              int window, int sink, int causal, void* stream) {
    FVK_CHECK(starts && new_lens && block_table && pages_held && free_pages && free_count && table_out && held_out && free_out && count_out && cu_q &&
                  kv_lens && granted, FVK_ERR_ARG, "fvk_paged_plan: null pointer");
    FVK_CHECK(n_requests >= 1 && n_requests <= PLAN_MAX_R, FVK_ERR_ARG, "fvk_paged_plan: n_requests=%d must be in 1..%d", n_requests, PLAN_MAX_R);
    FVK_CHECK(page_shift_of(page_size) >= 0, FVK_ERR_ARG, "fvk_paged_plan: page_size=%d must be 16, 32, 64, 128 or 256", page_size);
    FVK_CHECK(table_width >= 1 && n_free >= 1 && n_tokens >= 0, FVK_ERR_ARG, "fvk_paged_plan: table_width=%d n_free=%d n_tokens=%d", table_width, n_free, n_tokens);
    FVK_CHECK((long)table_width * page_size <= 0x7fffffffL && (long)n_requests * table_width <= 0x7fffffffL, FVK_ERR_ARG,
              "fvk_paged_plan: a table of %d x %d pages of %d tokens passes 32 bits", n_requests, table_width, page_size);
    FVK_CHECK(n_tokens == 0 || (slot_map && positions), FVK_ERR_ARG, "fvk_paged_plan: null slot_map / positions");
    FVK_CHECK(grid_h >= 1 && grid_w >= 1 && (long)grid_h * grid_w <= 0x7fffffffL, FVK_ERR_ARG, "fvk_paged_plan: grid %d x %d", grid_h, grid_w);
    FVK_CHECK(window >= 0 && sink >= 0 && (window > 0 || sink == 0), FVK_ERR_ARG, "fvk_paged_plan: window=%d sink=%d (a sink needs a window)", window, sink);
    FVK_CHECK(window == 0 || dead_counts, FVK_ERR_ARG, "fvk_paged_plan: a window needs dead_counts [2 * n_requests + 1]");
    // (many requests: every workgroup repeats their prefix sum, so fewer of them; 4096 rows of 200 cells take 62 us with a window, otherwise 141)
    const int row_waves = table_width > 64 && n_requests <= 1024 ? 4 : 1, table_blocks = (n_requests * row_waves + 3) / 4;
    const long items = n_tokens > n_free ? n_tokens : n_free;
    // one item per thread up to half a million of them: a second one waits for its request and page again (145 000 tokens: 8.8 us with four, 6.1 with one)
    const long per = n_requests <= 1024 ? 256 : 1024;
    const int blocks = (int)((items + per - 1) / per < 2048 ? (items + per - 1) / per : 2048);
    PlanArgs a{starts, new_lens, block_table, pages_held, free_pages, free_count, table_out, held_out, free_out, count_out, cu_q, kv_lens, slot_map,
               positions, granted, window > 0 ? dead_counts : nullptr, n_requests, table_width, n_free, page_size, n_tokens, grid_h, grid_w, window, sink,
               causal != 0, table_blocks, row_waves};
    hipLaunchKernelGGL(paged_plan_kernel, dim3(table_blocks + blocks), dim3(256), 0, (hipStream_t)stream, a);
    FVK_LAUNCH_CHECK();
    if (window > 0) {
        hipLaunchKernelGGL(paged_release_kernel, dim3((n_requests + 3) / 4), dim3(256), 0, (hipStream_t)stream, a);
        FVK_LAUNCH_CHECK();
    }
    return FVK_OK;
}

extern "C" int fvk_rmsnorm_rope_paged_bf16(const void* q, const void* k, const void* v, const void* wq, const void* wk, const int32_t* positions,
                                           const float* rope, const int32_t* slot_map, void* q_out, void* k_pages, void* v_pages, int T, int H, int Hkv,
                                           long q_stride, long k_stride, long v_stride, long out_stride, long k_page_stride, long k_row_stride,
                                           long k_head_stride, long v_page_stride, long v_row_stride, long v_head_stride, int n_pages, int page_size,
                                           int n_t, int n_h, int n_w, int dim_t, int dim_h, int dim_w, int round_norm, float eps, void* stream) {
    FVK_CHECK(q && k && v && slot_map && q_out && k_pages && v_pages, FVK_ERR_ARG, "fvk_rmsnorm_rope_paged_bf16: null pointer");
    FVK_CHECK(T >= 0 && H >= 1 && Hkv >= 1 && H <= 64 && Hkv <= 64, FVK_ERR_ARG, "fvk_rmsnorm_rope_paged_bf16: T=%d H=%d Hkv=%d (at most 64 heads)", T, H, Hkv);
    const int shift = page_shift_of(page_size);
    FVK_CHECK(shift >= 0 && n_pages >= 1 && (long)n_pages * page_size <= 0x7fffffffL, FVK_ERR_ARG,
              "fvk_rmsnorm_rope_paged_bf16: n_pages=%d page_size=%d (16, 32, 64, 128 or 256 tokens)", n_pages, page_size);
    // the stride of a dimension of one element says nothing
    if (T == 1) q_stride = k_stride = v_stride = out_stride = 0;
    if (Hkv == 1) k_head_stride = v_head_stride = 0;
    if (n_pages == 1) k_page_stride = v_page_stride = 0;
    FVK_CHECK(((q_stride | k_stride | v_stride | out_stride | k_page_stride | k_row_stride | k_head_stride | v_page_stride | v_row_stride | v_head_stride) & 7) == 0,
              FVK_ERR_ARG, "fvk_rmsnorm_rope_paged_bf16: strides must be multiples of 8 elements");
    FVK_CHECK((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)wq | (uintptr_t)wk) & 15) == 0,
              FVK_ERR_ARG, "fvk_rmsnorm_rope_paged_bf16: pointers must be 16-byte aligned");
    FVK_CHECK(!rope || (positions && n_t >= 1 && n_h >= 1 && n_w >= 1 && dim_t >= 0 && dim_h >= 0 && dim_w >= 0 && dim_t + dim_h + dim_w == 128 &&
                        dim_t % 2 == 0 && dim_h % 2 == 0), FVK_ERR_ARG,
              "fvk_rmsnorm_rope_paged_bf16: rotary table of %d x %d x %d positions over %d + %d + %d columns (even, 128 together)", n_t, n_h, n_w, dim_t, dim_h, dim_w);
    if (T == 0) return FVK_OK;
    int most = dim_t > dim_h ? dim_t : dim_h;
    most = most > dim_w ? most : dim_w;
    WriteArgs a{{(const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v}, {(const bf16_t*)wq, (const bf16_t*)wk}, positions, (const float2*)rope, slot_map,
                (bf16_t*)q_out, (bf16_t*)k_pages, (bf16_t*)v_pages, q_stride, k_stride, v_stride, out_stride, k_page_stride, k_row_stride, k_head_stride,
                v_page_stride, v_row_stride, v_head_stride, T, H, Hkv, most / 2, n_t, n_h, n_w, dim_t / 2, (dim_t + dim_h) / 2, shift, n_pages, round_norm != 0, eps};
    const int rc = dispatch_heads((H > Hkv ? H : Hkv) * 16, [&](auto vpl) {
        hipLaunchKernelGGL((rmsnorm_rope_paged_kernel<decltype(vpl)::value>), dim3((T + 3) / 4, 3), dim3(256), 0, (hipStream_t)stream, a);
        return FVK_OK;
    });
    FVK_CHECK(rc == FVK_OK, rc, "fvk_rmsnorm_rope_paged_bf16: unsupported H=%d", H);
    FVK_LAUNCH_CHECK();
    return FVK_OK;
}
