// Attention of a batch in which groups of sequences begin with the same pages: those are read and multiplied once for the whole group (fp16 cache, a
// query row per sequence and head).
//
//   y = softmax(q k^T / sqrt(d)) v over the positions 0 .. pos of a row.  With maximum m, sum of weights l and weighted values o of each part of the positions,
//   M = max m, y = sum o 2^(m - M) / sum l 2^(m - M): the parts are the pieces of the group's pages and the row's own ones.
//
// Two launches.  The first takes the groups' pages: the queries of all rows and of the heads of one key/value head stack on the rows of an MMA (row = sequence * heads + head), so
// that what every sequence alone would do bound by the cache's bytes, once per sequence, is a product of up to 256 rows by pages that are read once: tcgen05, as in
// attention_prefill_tc.cu, two tiles of 128 rows to a CTA, their steps of 128 tokens dealt out evenly to all SMs (a CTA's share may end in the middle of one
// key/value head and begin the next).  It leaves m, l and o of each piece.  The second launch takes the rows' own pages, a CTA (a cluster, where rows are few) for each row and
// key/value head, 16 tokens at a time on mma.sync, and joins them with the pieces; it is launched while the first one runs and waits for it ahead of the join.
//
// Both have queries and weights in fp16 (queries times a power of two of their row, so that any size goes in; weights at most 2^8), sums and maxima in f32: 2^-12 of a weight (of one below 2^-14 of
// the largest 2^-25 of that one's) is what a result is off by, at random, an eighth of the half step of a bf16 output.  Scores are f32 in the log2 domain: beyond its range, 2^128, a row is NaN.
//
// What bounds it (us of both launches, 32 heads of 128 on 8): 3 rows behind 16 pages 16 and 32 behind 250 with up to 300 tokens of their own 32 (the bytes 8): latencies one behind the other, of which the first
// launch has 6 us ahead of its first scores (places, plan, queries), a step's 1.0 to 1.8, 3 for sums on their way out, and the second one 5 for the join behind it.  200 behind 1000 with up to 400 of their own 147 (the
// products 66), and 174 once the card is at its power limit, after some 50 ms of nothing else (1545 MHz instead of 1965): a step of two tiles takes 1.8 us, of which the MMAs run 0.6: the chain scores,
// maximum, exponentials, weights of one tile is hidden by the other one's alone (more of the exponentials as polynomials: 154 to 158); the second launch reads the rows' own pages at 3.5 TB/s for 50 us, its
// CTAs of 200 tokens being starts and ends for the greater part.
#define WAIT_UNIT 5u
#include "attention_tc.cuh"
#include "epilogue.cuh"
#include "smem_limit.cuh"
#include "tensor_map.cuh"
#include "waits.cuh"

#define SH_PAGE 32
#define SH_ROWS 128                    // stacked rows of a tile
#define SH_KV 128                      // tokens of a step
#define SH_THREADS 384
#define SH_TILE_BYTES 32768            // 128 x 128 fp16
#define SH_STAGES 2
#define SH_OUT_LD 20
#define SH_MAX_GROUPS 8
#define SH_PAIR_COST 7                 // of a step with two tiles
#define SH_ONE_COST 4                  // ... with one
#define SH_LEAST_COST 8                // of a CTA's share: two steps of one tile
#define SH_BAD 8                       // items of a CTA that can be at work at once, and more
#define SH_FAR 0x1p20f                 // references in the log2 domain whose rounding shows in the weights
#define SH_OWN_TOK 16                  // tokens of a warp's turn
#define SH_OWN_MAX_CTAS 8

extern void dl_set_error(const char* fmt, ...);
extern int dl_device_sm_count();

struct ShArgs {
    const float* q;                    // [M][ldq]
    long long ldq;
    const __half *k_cache, *v_cache;   // [pages][n_kv][32][head size]
    const int *pos, *slot, *block_table, *groups;
    int M, n_heads, n_kv_heads, rep, n_slots, max_pages, n_pages, max_groups;      // rep: query heads of a key/value head
    uint8_t* scratch;                  // norms | sums
    int shares;                        // CTAs of the first launch
    long long n_pieces;                // that the scratch has room for
    uint8_t *xq_out, *xh_out;
    int out_mcap;
    void* y_out;
    long long ldy;
    int y_type;
};

// What the first launch works on.  Every CTA of both makes it for itself.
struct ShPlan {
    int n, quota;                                              // groups; a CTA's share
    int total;
    int begin[SH_MAX_GROUPS], end[SH_MAX_GROUPS];              // rows
    int pages[SH_MAX_GROUPS], first[SH_MAX_GROUPS];            // pages that all rows of the group see; a row whose table names them
    int cost[SH_MAX_GROUPS], unit[SH_MAX_GROUPS];              // cost and units (key/value head, two tiles) of the groups ahead
};

struct ShUnit { int g, kvh, pair, tiles, steps, w, c0, index; };

DL_DEVINL float2* sh_norms(const ShArgs& a) { return reinterpret_cast<float2*>(a.scratch); }                                 // [piece][2][128]
DL_DEVINL float4* sh_sums(const ShArgs& a) { return reinterpret_cast<float4*>(sh_norms(a) + a.n_pieces * 2 * SH_ROWS); }     // [piece][2][128][head size / 4]

// positions that a row sees; 0: it has no token, -1: its sequence or position is not in the table
DL_DEVINL int sh_tokens(const ShArgs& a, int m) {
    const int p = a.pos[m], s = a.slot[m];
    if (p < 0) return 0;
    return (unsigned)s < (unsigned)a.n_slots && p < a.max_pages * SH_PAGE ? p + 1 : -1;
}
// The list of groups, by the first threads of a CTA, into shared memory ([1 + 3 SH_MAX_GROUPS]; a barrier has to follow)
DL_DEVINL void sh_fetch_groups(const ShArgs& a, int* list) {
    const int i = threadIdx.x;
    if (i <= 3 * SH_MAX_GROUPS) list[i] = i <= 3 * a.max_groups ? a.groups[i] : 0;
}
// the rows of group i as they are taken: in order, none in two groups
DL_DEVINL void sh_group(const ShArgs& a, const int* list, int i, int& at, int& begin, int& end, int& pages) {
    begin = max(list[1 + 3 * i], at);
    end = min(list[2 + 3 * i], a.M);
    end = max(begin, end);
    pages = max(0, min(list[3 + 3 * i], a.max_pages));
    at = end;
}
DL_DEVINL int sh_n_groups(const ShArgs& a, const int* list) { return max(0, min(min(list[0], a.max_groups), SH_MAX_GROUPS)); }

DL_DEVINL int sh_tiles(const ShArgs& a, int rows) { return (rows * a.rep + SH_ROWS - 1) / SH_ROWS; }
DL_DEVINL int sh_steps(int pages) { return (pages + SH_KV / SH_PAGE - 1) / (SH_KV / SH_PAGE); }
// cost of a group's steps for one key/value head
DL_DEVINL int sh_head_cost(int tiles, int steps) { return steps * (tiles / 2 * SH_PAIR_COST + (tiles & 1) * SH_ONE_COST); }

DL_DEVINL void sh_unit(const ShArgs& a, const ShPlan& p, int g, int kvh, int pair, ShUnit& u) {
    const int tiles = sh_tiles(a, p.end[g] - p.begin[g]), pairs = (tiles + 1) / 2;
    u.g = g; u.kvh = kvh; u.pair = pair;
    u.tiles = min(2, tiles - 2 * pair);
    u.steps = sh_steps(p.pages[g]);
    u.w = u.tiles == 2 ? SH_PAIR_COST : SH_ONE_COST;
    u.c0 = p.cost[g] + kvh * sh_head_cost(tiles, u.steps) + pair * u.steps * SH_PAIR_COST;
    u.index = p.unit[g] + kvh * pairs + pair;
}
// x / d of numbers that are not negative, without the compiler's sequence for it (2000 clk of a CTA's start went there)
DL_DEVINL int sh_quot(int x, int d) {
    int q = (int)__fdividef((float)x, (float)d);
    while (q > 0 && (long long)q * d > x) q--;
    while ((long long)(q + 1) * d <= x) q++;
    return q;
}
// the unit in which place x of the whole cost lies
DL_DEVINL void sh_unit_at(const ShArgs& a, const ShPlan& p, int x, ShUnit& u) {
    int g = 0;
    while (g + 1 < p.n && p.cost[g + 1] <= x) g++;
    const int tiles = sh_tiles(a, p.end[g] - p.begin[g]), steps = sh_steps(p.pages[g]), head = sh_head_cost(tiles, steps), rest = x - p.cost[g];
    const int kvh = sh_quot(rest, head);
    sh_unit(a, p, g, kvh, min(sh_quot(rest - kvh * head, steps * SH_PAIR_COST), (tiles + 1) / 2 - 1), u);
}
// ... and the one behind it (there is one: the whole cost has not been reached)
DL_DEVINL void sh_next_unit(const ShArgs& a, const ShPlan& p, ShUnit& u) {
    int g = u.g, kvh = u.kvh, pair = u.pair + 1;
    if (pair * 2 >= sh_tiles(a, p.end[g] - p.begin[g])) { pair = 0; kvh++; }
    if (kvh == a.n_kv_heads) {
        kvh = 0;
        do g++; while (g + 1 < p.n && p.cost[g + 1] == p.cost[g]);      // (groups that cost nothing)
    }
    sh_unit(a, p, g, kvh, pair, u);
}
DL_DEVINL int sh_div(int x, int w) { return w == SH_PAIR_COST ? x / SH_PAIR_COST : x / SH_ONE_COST; }
// the steps [j0, j1) of a unit that share b has
DL_DEVINL void sh_share(const ShPlan& p, const ShUnit& u, int b, int& j0, int& j1) {
    const int lo = b * p.quota - u.c0, hi = lo + p.quota;
    j0 = lo <= 0 ? 0 : min(u.steps, sh_div(lo + u.w - 1, u.w));
    j1 = hi <= 0 ? 0 : min(u.steps, sh_div(hi + u.w - 1, u.w));
}

// the exponent field of the power of two that brings a row's largest value (its bits) to 2^8 .. 2^9; its inverse has 254 less that
DL_DEVINL unsigned sh_up(unsigned most) { return most == 0 ? 127u : min(262u - (most >> 23), 250u); }

// a barrier of the eight softmax warps
template <int ID> DL_DEVINL void sh_bar() { asm volatile("bar.sync %0, 256;" ::"n"(ID) : "memory"); }

struct ShItem {
    int kvh, row0, rows, begin, slot, pages, j0, J, tiles, piece;      // row0: first stacked row; rows: stacked rows of the group
    int number;                        // 1, 2, .. of the CTA's items
};

// Queries of 32 stacked rows into a tile's K-major, swizzled image; where one of them is beyond what fp16 holds well, each row times the power of two that brings its largest value to 2^8 .. 2^9
// (always, with a maximum over the warp for each row, the load took 5.3 us of a CTA's time).  Lane i holds the address of row r0 + i and gets what the scores of that row are multiplied with (NaN: the row is not finite).
template <int HS, typename Ready>
DL_DEVINL float sh_load_rows(const float* mine, uint8_t* tile, int r0, Ready ready) {
    constexpr int PER = 128 / HS;                              // rows a load
    const int lane = threadIdx.x & 31, in = lane * 4 / HS, col = lane * 4 % HS;
    uint8_t* qd = tile + (r0 + in) * 128 + (col >> 6) * 16384 + (lane & 1) * 8;
    constexpr int BATCH = 16;                                    // (a loop: all 32 rows side by side are code that every launch reads anew, 11 rows behind a book 44.2 us instead of 42.3)
    float factor = 1.f;
    // rows whose largest value is 2^-6 or more and below 2^15, as queries are, go in as they are (a NaN, too: its row's scores are NaN)
    unsigned large = 0;                                          // a bit for each row of which this lane has such a value
    float top = 0.f;
#pragma unroll 1
    for (int u0 = 0; u0 < 32; u0 += BATCH) {
        float4 x[BATCH / PER];
#pragma unroll
        for (int u = 0; u < BATCH; u += PER) {
            const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)mine, u0 + u + in)) + col;
            x[u / PER] = *reinterpret_cast<const float4*>(src);
        }
        if (u0 == 0) ready();
#pragma unroll
        for (int u = 0; u < BATCH; u += PER) {                    // 16-byte piece c of a half row -> swizzled slot c ^ (row & 7)
            const float4& y = x[u / PER];
            const float most = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
            top = fmaxf(top, most);
            large |= most >= 0x1p-6f ? 1u << (u0 + u) : 0u;
            *reinterpret_cast<uint2*>(qd + (u0 + u) * 128 + ((((lane >> 1) & 7) ^ ((u + in) & 7)) << 4)) = make_uint2(pt_pack2<false>(y.x, y.y), pt_pack2<false>(y.z, y.w));
        }
    }
    large <<= in;
    const bool plain = __reduce_or_sync(0xffffffffu, large) == 0xffffffffu && __reduce_max_sync(0xffffffffu, __float_as_uint(top)) < 0x47000000u;
    if (!plain) {
#pragma unroll 1
        for (int u = 0; u < 32; u += PER) {
            const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)mine, u + in)) + col);
            unsigned most = max(max(__float_as_uint(y.x) & 0x7fffffffu, __float_as_uint(y.y) & 0x7fffffffu), max(__float_as_uint(y.z) & 0x7fffffffu, __float_as_uint(y.w) & 0x7fffffffu));
#pragma unroll
            for (int o = HS / 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const bool finite = most < 0x7f800000u;
            const unsigned up = sh_up(most);
            const float by = finite ? __uint_as_float(up << 23) : 0.f, back = finite ? __uint_as_float((254u - up) << 23) : __uint_as_float(0x7fffffffu);
            // (an infinity or NaN times zero is a NaN, in its row alone)
            *reinterpret_cast<uint2*>(qd + u * 128 + ((((lane >> 1) & 7) ^ ((u + in) & 7)) << 4)) = make_uint2(pt_pack2<false>(y.x * by, y.y * by), pt_pack2<false>(y.z * by, y.w * by));
            const float row = __shfl_sync(0xffffffffu, back, lane % PER * (HS / 4));
            if (lane / PER * PER == u) factor = row;
        }
    }
    fence_proxy_async_smem();
    return factor;
}

// The plan, by all threads of a CTA (in shared memory).
DL_DEVINL void sh_make_plan(const ShArgs& a, ShPlan& p, int* list, int (*red)[2]) {
    const int tid = threadIdx.x;
    const int n_thr = blockDim.x;
    int mine[4];                                                 // (asked for together with the list)
#pragma unroll
    for (int i = 0; i < 4; i++) mine[i] = tid + i * n_thr < a.M ? sh_tokens(a, tid + i * n_thr) : 0;
    sh_fetch_groups(a, list);
    if (tid < 2 * SH_MAX_GROUPS) red[tid >> 1][tid & 1] = 0x7fffffff;
    __syncthreads();
    const int n = sh_n_groups(a, list);
    int at = 0, b, e, pages;
    for (int g = 0; g < n; g++) {
        sh_group(a, list, g, at, b, e, pages);
        int least = 0x7fffffff, first = 0x7fffffff;
        auto see = [&](int m, int t) {
            if (m >= b && m < e && t > 0) { least = min(least, t / SH_PAGE); first = min(first, m); }
        };
#pragma unroll
        for (int i = 0; i < 4; i++) see(tid + i * n_thr, mine[i]);
        for (int m = tid + 4 * n_thr; m < e; m += n_thr)
            if (m >= b) see(m, sh_tokens(a, m));
        least = __reduce_min_sync(0xffffffffu, least);
        first = __reduce_min_sync(0xffffffffu, first);
        if ((tid & 31) == 0 && first != 0x7fffffff) { atomicMin(&red[g][0], least); atomicMin(&red[g][1], first); }
    }
    __syncthreads();
    if (tid == 0) {
        int unit = 0, cost = 0;
        at = 0;
        for (int g = 0; g < n; g++) {
            sh_group(a, list, g, at, b, e, pages);
            pages = red[g][1] == 0x7fffffff ? 0 : min(pages, red[g][0]);
            const int tiles = sh_tiles(a, e - b);
            p.begin[g] = b; p.end[g] = e; p.pages[g] = pages; p.first[g] = red[g][1]; p.cost[g] = cost; p.unit[g] = unit;
            cost += a.n_kv_heads * sh_head_cost(tiles, sh_steps(pages));      // (the host has seen to it that all of it fits)
            unit += a.n_kv_heads * ((tiles + 1) / 2);
        }
        p.n = n;
        p.total = cost;
        p.quota = max(sh_quot(cost + a.shares - 1, a.shares), SH_LEAST_COST);
    }
    __syncthreads();
}

template <int HS>
__global__ void __launch_bounds__(SH_THREADS, 1) shared_attention_kernel(const __grid_constant__ ShArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                         const __grid_constant__ WaitLimit limit) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ ShPlan plan;
    __shared__ int list[1 + 3 * SH_MAX_GROUPS], red[SH_MAX_GROUPS][2], gave_up_s, bad_s[SH_BAD];      // bad_s: the number of an item with a page that is none, at its place modulo SH_BAD
    uint8_t* q_s = smem;                                        // [2] query tiles
    uint8_t* k_s = q_s + 2 * SH_TILE_BYTES;                     // [2] K tiles (tokens x head dim, K-major)
    uint8_t* v_s = k_s + SH_STAGES * SH_TILE_BYTES;             // [2] V tiles (tokens x head dim, MN-major for P V)
    __shared__ float2 ml_s[SH_ROWS];                            // maxima and sums of the second place
    float* out_s = reinterpret_cast<float*>(v_s + SH_STAGES * SH_TILE_BYTES);      // [8 warps][32][SH_OUT_LD] f32: sums on their way out
    uint64_t* bars = reinterpret_cast<uint64_t*>(out_s + 8 * 32 * SH_OUT_LD);
    uint64_t* k_full = bars;             // [2] transaction bytes of the step's K copies
    uint64_t* k_empty = bars + 2;        // [2] the scores that read the stage are complete (both tiles')
    uint64_t* v_full = bars + 4;         // [2] transaction bytes of the step's V copies
    uint64_t* v_empty = bars + 6;        // [2] P V of the step has retired (both tiles')
    uint64_t* q_full = bars + 8;         // [2] the tile's queries are there
    uint64_t* q_empty = bars + 10;       // [2] the tile's last scores are complete
    uint64_t* s_full = bars + 12;        // [2] scores complete
    uint64_t* p_full = bars + 14;        // [2] probabilities written
    uint64_t* o_full = bars + 16;        // [2] P V complete
    uint64_t* s_empty = bars + 18;       // the scores have been read into registers (one buffer for both tiles)
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 19);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        gave_up_s = limit.ns == 0;
        for (int i = 0; i < SH_BAD; i++) bad_s[i] = 0;
        for (int s = 0; s < 2; s++) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
            mbar_init(&q_full[s], 128);
            mbar_init(&q_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 128);
            mbar_init(&o_full[s], 1);
        }
        mbar_init(s_empty, 128);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(tmem_holder, 512);                 // (ahead of the wait: the block has the SM's registers, so that nothing it waits for can want tensor memory beside it)
    pdl_wait();                                                  // q, the rows' places and the cache come from earlier kernels
    pdl_launch_dependents();                                     // ... and are complete for the second launch, too, when it starts
    sh_make_plan(a, plan, list, red);
    const int b = blockIdx.x, x_end = min((int)min((long long)plan.total, (long long)(b + 1) * plan.quota), plan.total);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if ((long long)b * plan.quota >= plan.total) {               // (uniform for the CTA)
        if (warp == 0) tmem_dealloc(__shfl_sync(0xffffffffu, *tmem_holder, 0), 512);
        return;
    }
    const PtWaits wait = {&gave_up_s, globaltimer_ns(), limit.ns};
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_holder, 0);
    // this CTA's items, in the same order for every role: `x` goes from the start of its share to the end of the unit looked at
    ShUnit u_at;
    int n_items = 0;
    auto next_item = [&](int& x, ShItem& it) {
        while (x < x_end) {
            int j0, j1;
            if (x == b * plan.quota) sh_unit_at(a, plan, x, u_at);
            else sh_next_unit(a, plan, u_at);
            sh_share(plan, u_at, b, j0, j1);
            x = u_at.c0 + u_at.steps * u_at.w;
            if (j1 <= j0) continue;
            it.kvh = u_at.kvh;
            it.begin = plan.begin[u_at.g];
            it.row0 = u_at.pair * 2 * SH_ROWS;
            it.rows = (plan.end[u_at.g] - it.begin) * a.rep;
            it.slot = plan.first[u_at.g];
            it.pages = plan.pages[u_at.g];
            it.j0 = j0;
            it.J = j1 - j0;
            it.tiles = u_at.tiles;
            it.piece = u_at.index + b;
            it.number = ++n_items;
            return true;
        }
        return false;
    };
    // A single tile takes both places, too: its steps in turn, so that the softmax of one step runs beside the next one's (a step took 1.9 us in one place, 1.6 for two tiles).
    // TMEM columns: one buffer of scores at 0, which the tiles take in turn; probabilities at 128, of 64 columns for each tile; outputs at 256 + 128 t
    if (warp < 8) {
        // ---------------- softmax: warps 0-3 tile 0, warps 4-7 tile 1; a thread per stacked row (= TMEM lane) ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, rep = a.rep;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16, T_S = tmem_base + lane_base, T_P = tmem_base + lane_base + 128 + t * 64, T_O = tmem_base + lane_base + 256 + t * 128;
        uint32_t ns = 0, nq = 0;                                 // steps of this tile so far, items whose queries are loaded
        float q_factor = 1.f;
        auto load_queries = [&](const ShItem& of) {
            if (of.tiles == 1 && of.J <= t) return;
            const int r = min(of.row0 + (of.tiles == 2 ? t * SH_ROWS : 0) + row, of.rows - 1);      // rows that are not there: the last one
            const int of_row = sh_quot(r, rep);
            q_factor = sh_load_rows<HS>(a.q + (long long)(of.begin + of_row) * a.ldq + (of.kvh * rep + r - of_row * rep) * HS, q_s + t * SH_TILE_BYTES, quarter * 32, [&] {
                if (nq > 0) wait(&q_empty[t], (nq - 1) & 1);      // the tile's last scores have read the queries before
            });
            nq++;
            mbar_arrive(&q_full[t]);
        };
        ShItem it{}, next{};                                     // (first an item without steps, so that the code for the next one's queries stands here once)
        int x = b * plan.quota;
        for (bool more = true; more; it = next) {
            const int by = it.tiles == 2 ? 1 : 2, ja = it.tiles == 2 ? 0 : t;      // steps ja, ja + by .. are this place's
            const float sc = 1.4426950408889634f * rsqrtf((float)HS) * q_factor;      // scores in the log2 domain
            float m_used = -INFINITY, l = 0.f;
            for (int j = ja; j < it.J; j += by, ns++) {
                uint32_t v[4][32];
                wait(&s_full[t], ns & 1);
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld_32x32b_x32(T_S + c * 32, v[c]);
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(s_empty);                            // the next scores may take the place
                const int lim = it.pages - (it.j0 + j) * (SH_KV / SH_PAGE);      // pages of this step
                if (lim < SH_KV / SH_PAGE) {
#pragma unroll
                    for (int c = 1; c < 4; c++)
                        if (c >= lim) {
#pragma unroll
                            for (int e = 0; e < 32; e++) v[c][e] = 0xff800000u;        // -inf
                        }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; e += 2)
#pragma unroll
                    for (int c = 0; c < 4; c++) mx4[c] = pt_max<true>(mx4[c], pt_max<true>(__uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1])));
                const float mx = pt_max<true>(pt_max<true>(mx4[0], mx4[1]), pt_max<true>(mx4[2], mx4[3])) * sc;
                // the reference may lag the maximum by 2^8; a NaN makes it NaN, and with it the sum of the weights for good
                const bool need = !(mx <= m_used || mx - m_used <= 8.0f);
                const bool moved = __any_sync(0xffffffffu, need);
                float alpha = 1.f;
                if (moved) {
                    const float m_new = need ? mx : m_used;
                    if (need) alpha = pt_ex2(m_used - m_new);
                    l *= alpha;
                    m_used = m_new;
                }
                const float ref = (m_used == -INFINITY) ? 0.0f : m_used;
                float by = sc, from = ref;
                if (__any_sync(0xffffffffu, fabsf(ref) >= SH_FAR)) {
                    // the exact product less a rounded one leaves the largest score that rounding for an exponent (from 2^28 on up to 16 either way: a weight beyond fp16, or next to
                    // none): the rounded products, as the maximum was formed
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int e = 0; e < 32; e++) v[c][e] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(v[c][e]), sc), ref));
                    by = 1.f;
                    from = 0.f;
                }
                pair_f sum = 0;
                uint32_t pk[4][16], none[1];
                if (j > ja) wait(&o_full[t], (ns - 1) & 1);
                tc_fence_after();
                if (moved && j > ja) {      // the accumulated output moves to the new reference (rare after the first steps)
                    uint32_t w[32];
#pragma unroll 1
                    for (int ch = 0; ch < HS / 32; ch++) {
                        tmem_ld_32x32b_x32(T_O + ch * 32, w);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) w[e] = __float_as_uint(__uint_as_float(w[e]) * alpha);
                        tmem_st_32x32b_x32(T_O + ch * 32, w);
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    pt_probs<false>(v[c], by, from, pk[c], none, sum);
                    tmem_st_32x32b_x16(T_P + c * 16, pk[c]);
                }
                l += pair_sum(sum);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            more = next_item(x, next);
            if (more) load_queries(next);
            if (ja >= it.J) continue;
            wait(&o_full[t], (ns - 1) & 1);
            tc_fence_after();
            // the largest weight is 1 or more; where it is not, a score was no number.  No score at all above -inf: nothing to add
            l = m_used == -INFINITY ? 0.f : l >= 0x1p-13f ? l : __int_as_float(0x7fffffff);
            if (*(volatile int*)&bad_s[it.number % SH_BAD] == it.number || gave_up_s) l = __int_as_float(0x7fffffff);
            // the two places of one tile have seen different steps of the same rows: the first one joins them (both lie in the same lanes of tensor memory)
            const bool pair = it.tiles == 1 && it.J > 1;
            float e0 = 1.f, e1 = 0.f;
            if (pair) {
                if (t == 1) {
                    ml_s[row] = make_float2(m_used, l);
                    tc_fence_before();
                    sh_bar<1>();                                 // place 1 is complete
                    sh_bar<2>();                                 // ... and read
                    continue;
                }
                sh_bar<1>();
                tc_fence_after();
                const float2 o1 = ml_s[row];
                const float top = fmaxf(l != 0.f ? m_used : -INFINITY, o1.y != 0.f ? o1.x : -INFINITY), ref = top == -INFINITY ? 0.f : top;
                e0 = l != 0.f ? pt_ex2(m_used - ref) : 0.f;
                e1 = o1.y != 0.f ? pt_ex2(o1.x - ref) : 0.f;
                l = l * e0 + o1.y * e1;
                m_used = top;
            }
            const size_t at = (size_t)it.piece * 2 + t;
            sh_norms(a)[at * SH_ROWS + row] = make_float2(m_used, l);
            // 16 columns of the warp's rows at a time, then as many lanes along a row (a thread along its own row: 5 us for 128 of them)
            float4* out = sh_sums(a) + (at * SH_ROWS + quarter * 32) * (HS / 4);
            float* stage = out_s + (size_t)warp * 32 * SH_OUT_LD;
            const int live = it.rows - (it.row0 + (it.tiles == 2 ? t * SH_ROWS : 0) + quarter * 32);      // rows of this warp that are there
#pragma unroll 1
            for (int ch = 0; ch < HS / 16; ch++) {
                uint32_t o[16], p[16];
                tmem_ld_32x32b_x16(T_O + ch * 16, o);
                if (pair) tmem_ld_32x32b_x16(T_O + 128 + ch * 16, p);
                tmem_ld_wait();
                if (pair) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {               // (a place in which nothing was seen may hold anything)
                        const float x = e0 != 0.f ? __uint_as_float(o[e]) * e0 : 0.f;
                        o[e] = __float_as_uint(e1 != 0.f ? fmaf(__uint_as_float(p[e]), e1, x) : x);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(stage + lane * SH_OUT_LD + e) = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                __syncwarp();
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += 8) {
                    const int r = r0 + (lane >> 2);
                    if (r < live) out[r * (HS / 4) + ch * 4 + (lane & 3)] = *reinterpret_cast<const float4*>(stage + r * SH_OUT_LD + (lane & 3) * 4);
                }
            }
            tc_fence_before();                                   // the next item's P V may write the output (behind p_full)
            if (pair) sh_bar<2>();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
        // The two products have a warp each: what one of them waits for does not hold up the other's (by one warp, scores behind the weights two steps ahead of them, a step of two tiles took 2.2 us).
        // What is multiplied, in this order: (place, step) (0, 0), (1, 0), (0, 1) .. of two tiles, (0, 0), (1, 1), (0, 2) .. of one
        if (warp == 8) {
            // ---------------- S = Q K^T ----------------
            const uint32_t idesc_s = pt_idesc(SH_ROWS, SH_KV, 0, false);
            const uint32_t q_lo = ((smem_u32(q_s) & 0x3FFFFu) >> 4) | (1u << 16), k_lo = ((smem_u32(k_s) & 0x3FFFFu) >> 4) | (1u << 16);
            uint32_t g = 0, q_phase = 0, s_phase = 1;            // steps so far; parities of q_full (a bit for each place) and s_empty (which is free at first)
            ShItem it;
            for (int x = b * plan.quota; next_item(x, it);) {
                auto scores = [&](int t, int st, bool first, bool last) {
                    if (first) {
                        wait(&q_full[t], q_phase >> t & 1);
                        q_phase ^= 1u << t;
                    }
                    wait(s_empty, s_phase);
                    s_phase ^= 1;
                    tc_fence_after();
                    __syncwarp();
                    if constexpr (HS == 128) pt_mma_ss(tmem_base, q_lo + t * (SH_TILE_BYTES >> 4), k_lo + st * (SH_TILE_BYTES >> 4), desc_hi, idesc_s, 0);
                    else pt_mma_ss4(tmem_base, q_lo + t * (SH_TILE_BYTES >> 4), k_lo + st * (SH_TILE_BYTES >> 4), desc_hi, idesc_s, 0);
                    pt_commit(&s_full[t]);
                    if (last) pt_commit(&q_empty[t]);
                };
                for (int j = 0; j < it.J; j++, g++) {
                    const int st = g & 1;
                    wait(&k_full[st], (g >> 1) & 1);
                    if (it.tiles == 2) {
                        scores(0, st, j == 0, j + 1 == it.J);
                        scores(1, st, j == 0, j + 1 == it.J);
                    } else scores(j & 1, st, j < 2, j + 2 >= it.J);
                    pt_commit(&k_empty[st]);
                }
            }
        } else if (warp == 11) {
            // ---------------- O += P V ----------------
            const uint32_t idesc_pv = pt_idesc(SH_ROWS, HS, 1, false);
            const uint32_t v_lo = ((smem_u32(v_s) & 0x3FFFFu) >> 4) | ((16384u >> 4) << 16);
            uint32_t g = 0, p_phase = 0;                         // steps so far, parities of p_full
            ShItem it;
            for (int x = b * plan.quota; next_item(x, it);) {
                auto weigh = [&](int t, int st, bool first) {
                    wait(&p_full[t], p_phase >> t & 1);
                    p_phase ^= 1u << t;
                    tc_fence_after();
                    __syncwarp();
                    pt_mma_ts(tmem_base + 256 + t * 128, tmem_base + 128 + t * 64, v_lo + st * (SH_TILE_BYTES >> 4), desc_hi, idesc_pv, first ? 0u : 1u);
                    pt_commit(&o_full[t]);
                };
                for (int j = 0; j < it.J; j++, g++) {
                    const int st = g & 1, live = it.pages - (it.j0 + j) * (SH_KV / SH_PAGE);
                    wait(&v_full[st], (g >> 1) & 1);
                    if (live < SH_KV / SH_PAGE) {                // pages that were not copied: a weight of zero times what lies there may be a NaN
                        uint8_t* vz = v_s + st * SH_TILE_BYTES;
                        for (int i = live * SH_PAGE * (HS / 8) + lane; i < SH_KV * (HS / 8); i += 32) {      // 16-byte pieces of a token's row
                            const int r = i / (HS / 8), c = i % (HS / 8);
                            *reinterpret_cast<uint4*>(vz + (c >> 3) * 16384 + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (it.tiles == 2) {
                        weigh(0, st, j == 0);
                        weigh(1, st, j == 0);
                    } else weigh(j & 1, st, j < 2);
                    pt_commit(&v_empty[st]);
                }
            }
        } else if (warp == 9 || warp == 10) {
            // ---------------- K producer (warp 9) / V producer (warp 10): a lane for each of a step's four pages ----------------
            const bool is_k = warp == 9;
            const uint64_t map = is_k ? reinterpret_cast<uint64_t>(&kmap) : reinterpret_cast<uint64_t>(&vmap);
            uint64_t* full = is_k ? k_full : v_full;
            uint64_t* empty = is_k ? k_empty : v_empty;
            uint8_t* ring = is_k ? k_s : v_s;
            uint32_t g = 0;
            ShItem it;
            for (int x = b * plan.quota; next_item(x, it);) {
                const int* bt = a.block_table + (size_t)a.slot[it.slot] * a.max_pages;
                const int last = min(it.pages, 4 * (it.j0 + it.J));      // pages of this item end here
                auto page_of = [&](int p) {                      // (not in the cache: the first one, and the piece is not valid)
                    if (lane >= 4 || p >= last) return -1;
                    const int page = bt[p];
                    if ((unsigned)page < (unsigned)a.n_pages) return page;
                    *(volatile int*)&bad_s[it.number % SH_BAD] = it.number;      // (seen by the softmax threads behind the barriers; another item's rows keep their values)
                    return 0;
                };
                auto line_of = [&](int page) { return (page * a.n_kv_heads + it.kvh) * SH_PAGE; };      // first row of the page in the [rows][head size] view
                int next = page_of(4 * it.j0 + lane);
                for (int j = 0; j < it.J; j++, g++) {
                    const int st = g & 1, page = next;
                    next = page_of(4 * (it.j0 + j + 1) + lane);  // (a step ahead, so that the table's latency is not in the copies' way)
                    if (g >= SH_STAGES) wait(&empty[st], ((g >> 1) & 1) ^ 1);
                    if (__any_sync(0xffffffffu, gave_up_s)) break;      // no more copies into a CTA that ends
                    if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)min(4, last - 4 * (it.j0 + j)) * (HS / 64) * 4096u);
                    __syncwarp();
                    if (page >= 0) {
                        const uint32_t dst = smem_u32(ring + st * SH_TILE_BYTES) + lane * 4096, bar = smem_u32(&full[st]);
#pragma unroll
                        for (int h = 0; h < HS / 64; h++)
                            asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst + h * 16384), "l"(map), "r"(h * 64),
                                         "r"(line_of(page)), "r"(bar)
                                         : "memory");
                    }
                    __syncwarp();
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (gave_up_s) {
        if (tid == 0) wait_report(limit);
        wait_settle();
    }
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ------------------------------------------------------------------------------------------------
// the rows' own pages, and the join
// ------------------------------------------------------------------------------------------------
DL_DEVINL void sh_cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
DL_DEVINL void sh_ldm(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
DL_DEVINL void sh_ldm_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
DL_DEVINL void sh_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// grid (CTAs of a row's cluster, key/value heads, rows).  Rows of the MMAs: the query heads of the key/value head (16 at most); tokens 16 at a time, a ring of stages for each
// warp.  Then every thread joins four values of a head over the warps and this CTA's pieces, and the cluster's CTAs over each other's.
template <int HS, int WARPS, int HALVES>
__global__ void __launch_bounds__(WARPS * 32, 12 / WARPS) shared_own_kernel(const __grid_constant__ ShArgs a) {
    constexpr int ROWB = HS * 2, CH = ROWB / 16, HALF = SH_OWN_TOK * ROWB, ST = 256 / HS;      // bytes and 16-byte pieces of a line, bytes of a turn's K or V, stages
    constexpr int KS = HS / 16, NT = HS / 8, LPH = HS / 4;                                     // MMA steps of a score, tiles of an output, threads of a head in the join
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ ShPlan plan;
    __shared__ int list[1 + 3 * SH_MAX_GROUPS], red[SH_MAX_GROUPS][2], bad_s;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x, n_cl = gridDim.x, kvh = blockIdx.y, m = blockIdx.z;           // (a row of the grid is one cluster)
    const int G = a.rep;
    float* w_acc = reinterpret_cast<float*>(smem);              // [warps][G][HS], after the ring is done with
    float* w_ml = w_acc + WARPS * G * HS;                // [warps][G][2]
    float* c_acc = w_ml + WARPS * G * 2;                 // [G][HS] of the CTA
    float* c_ml = c_acc + G * HS;                               // [G][2]
    pdl_launch_dependents();
    if (tid == 0) bad_s = 0;
    const int g = lane >> 2, qd = lane & 3;
    // what needs no more than the row's number is asked for at once: its place, its queries (head g, and g + 8 where there are so many), and what the plan is made of
    const int T = sh_tokens(a, m), slot = a.slot[m];
    float2 qx[HALVES][KS][2];
#pragma unroll
    for (int u = 0; u < HALVES; ++u) {
        const int h = g + u * 8;
        const float* q = a.q + (long long)m * a.ldq + (size_t)(kvh * G + (h < G ? h : 0)) * HS + qd * 2;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int w = 0; w < 2; ++w) qx[u][k][w] = *reinterpret_cast<const float2*>(q + k * 16 + w * 8);
    }
    sh_make_plan(a, plan, list, red);
    int g_of = -1;                                               // the row's group, and the pages that all of its rows see
    for (int i = 0; i < plan.n; i++)
        if (m >= plan.begin[i] && m < plan.end[i]) { g_of = i; break; }
    const int shared = g_of >= 0 ? plan.pages[g_of] : 0;
    const int n_pages = T > 0 ? (T + SH_PAGE - 1) / SH_PAGE : 0;
    const int own = T > 0 ? n_pages - shared : 0, shares = max(1, min(n_cl, (own + 7) / 8)), per = (own + shares - 1) / shares;
    const int pg0 = shared + min(own, rank * per), pg1 = shared + (rank < shares ? min(own, rank * per + per) : 0);
    const int t_end = min(max(T, 0), pg1 * SH_PAGE);
    const int n_turns = pg1 > pg0 ? (t_end - pg0 * SH_PAGE + SH_OWN_TOK - 1) / SH_OWN_TOK : 0, n_my = (n_turns - warp + WARPS - 1) / WARPS;      // warp w takes turns w, w + 4, ...
    const int* bt = a.block_table + (size_t)(T > 0 ? slot : 0) * a.max_pages;
    const uint32_t ring = smem_u32(smem) + warp * (ST * 2 * HALF);
    float run_m[HALVES], run_l[HALVES];                          // of heads g and g + 8; run_l: this lane's own tokens
#pragma unroll
    for (int u = 0; u < HALVES; ++u) { run_m[u] = -INFINITY; run_l[u] = 0.f; }
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    bool bad = false;
    if (n_my > 0) {
        auto page_at = [&](int i) {
            if (i >= n_my) return 0;
            const int p = bt[pg0 + ((warp + WARPS * i) >> 1)];
            if ((unsigned)p < (unsigned)a.n_pages) return p;
            bad = true;
            return 0;
        };
        int my_page = page_at(lane);                             // the lanes hold the next 32 turns' page numbers
        const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.k_cache), *vc = reinterpret_cast<const uint8_t*>(a.v_cache);
        auto load = [&](int i, int st, int page) {
            const int turn = warp + WARPS * i;
            const int left = t_end - pg0 * SH_PAGE - turn * SH_OWN_TOK;      // tokens from this turn on
            const size_t off = (((size_t)page * a.n_kv_heads + kvh) * SH_PAGE + (turn & 1) * SH_OWN_TOK) * (size_t)ROWB;
            const uint32_t dst = ring + st * (2 * HALF);
#pragma unroll
            for (int j = 0; j < SH_OWN_TOK * CH / 32; ++j) {
                const int idx = j * 32 + lane, t = idx / CH, c = idx % CH;
                const uint32_t d = dst + t * ROWB + ((c ^ (t & 7)) << 4);
                sh_cp16(d, kc + off + (size_t)idx * 16, t < left);
                sh_cp16(d + HALF, vc + off + (size_t)idx * 16, t < left);
            }
        };
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) {
            const int page = __shfl_sync(0xffffffffu, my_page, i);
            if (i < n_my) load(i, i, page);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        // queries in the A fragments: head g in rows g, head g + 8 in rows g + 8; times a power of two of the head
        uint32_t qf[KS][4];
        float sc[HALVES];
        if (HALVES == 1)
#pragma unroll
            for (int k = 0; k < KS; ++k) qf[k][1] = qf[k][3] = 0u;
#pragma unroll
        for (int u = 0; u < HALVES; ++u) {
            sc[u] = 0.f;
            unsigned most = 0;
            const float2 (&x)[KS][2] = qx[u];
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int w = 0; w < 2; ++w) most = max(most, max(__float_as_uint(x[k][w].x) & 0x7fffffffu, __float_as_uint(x[k][w].y) & 0x7fffffffu));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const bool finite = most < 0x7f800000u, there = g + u * 8 < G;
            const unsigned up = sh_up(most);
            const float by = finite && there ? __uint_as_float(up << 23) : 0.f;
            sc[u] = (finite ? __uint_as_float((254u - up) << 23) : __uint_as_float(0x7fffffffu)) * (1.44269504088896341f * rsqrtf((float)HS));
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int w = 0; w < 2; ++w) qf[k][2 * w + u] = there ? pt_pack2<false>(x[k][w].x * by, x[k][w].y * by) : 0u;
        }
        int st = 0;
        for (int i = 0; i < n_my; ++i) {
            {
                const int nx = i + ST - 1;
                if ((nx & 31) == 0) my_page = page_at(nx + lane);
                const int page = __shfl_sync(0xffffffffu, my_page, nx & 31);
                if (nx < n_my) load(nx, st == 0 ? ST - 1 : st - 1, page);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
            __syncwarp();
            const uint32_t kb = ring + st * (2 * HALF), vb = kb + HALF;
            float c[2][4] = {};                                  // n-tile j = tokens 8 j ..
            {
                const int t = (lane & 7) + ((lane >> 4) << 3), c1 = (lane >> 3) & 1;
                const uint32_t base = kb + t * ROWB;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t b[4];
                    sh_ldm(b, base + (((2 * k + c1) ^ (t & 7)) << 4));
                    sh_mma(c[0], qf[k], b[0], b[1]);
                    sh_mma(c[1], qf[k], b[2], b[3]);
                }
            }
            const int left = t_end - pg0 * SH_PAGE - (warp + WARPS * i) * SH_OWN_TOK;
            uint32_t pa[4] = {0u, 0u, 0u, 0u};
            float corr[HALVES];
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                float mx = -INFINITY, s[2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = c[j][2 * u + e] * sc[u];
                        s[j][e] = (j * 8 + qd * 2 + e < left) ? v : -INFINITY;
                        mx = fmaxf(mx, s[j][e]);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float m_new = fmaxf(run_m[u], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
                corr[u] = pt_ex2(run_m[u] - m_use);
                run_m[u] = m_new;
                float ps = 0.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p0 = pt_ex2(s[j][0] - m_use), p1 = pt_ex2(s[j][1] - m_use);
                    ps += p0 + p1;
                    pa[2 * j + u] = pt_pack2<false>(p0, p1);
                }
                run_l[u] = fmaf(run_l[u], corr[u], ps);
            }
            {
                const int t = (lane & 7) + (((lane >> 3) & 1) << 3), c1 = lane >> 4;
                const uint32_t base = vb + t * ROWB;
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b[4];
                    sh_ldm_trans(b, base + (((n + c1) ^ (t & 7)) << 4));
#pragma unroll
                    for (int e = 0; e < 2 * HALVES; ++e) { o[n][e] *= corr[e >> 1]; o[n + 1][e] *= corr[e >> 1]; }
                    sh_mma(o[n], pa, b[0], b[1]);
                    sh_mma(o[n + 1], pa, b[2], b[3]);
                }
            }
            __syncwarp();
            st = st == ST - 1 ? 0 : st + 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
#pragma unroll
    for (int u = 0; u < HALVES; ++u) {
        run_l[u] += __shfl_xor_sync(0xffffffffu, run_l[u], 1);
        run_l[u] += __shfl_xor_sync(0xffffffffu, run_l[u], 2);
    }
    if (bad) bad_s = 1;
    __syncthreads();                                             // the rings are done with
#pragma unroll
    for (int u = 0; u < HALVES; ++u) {
        const int h = g + u * 8;
        if (h >= G) continue;
        float* w = w_acc + (warp * G + h) * HS + qd * 2;
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(w + n * 8) = make_float2(o[n][2 * u], o[n][2 * u + 1]);
        if (qd == 0) { w_ml[(warp * G + h) * 2] = run_m[u]; w_ml[(warp * G + h) * 2 + 1] = run_l[u]; }
    }
    pdl_wait();                                                  // the pieces (and what follows this launch follows the first one, too)
    __syncthreads();
    // A warp joins a head, a lane four of its values (heads of 64: half a warp every other piece): the warps' own parts, then this CTA's pieces of the group's pages (those of every n_cl-th share),
    // 32 maxima and sums at a time, and their values all in flight.
    for (int h = warp; h < G; h += WARPS) {
        const int d4 = lane % LPH, half = lane / LPH;
        float M = -INFINITY, L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        auto put = [&](const float4& x, float e) { O = make_float4(fmaf(x.x, e, O.x), fmaf(x.y, e, O.y), fmaf(x.z, e, O.z), fmaf(x.w, e, O.w)); };
        // maxima and sums of 32 parts (sum 0: nothing was seen; a NaN is something), one a lane: this lane's factor
        auto weigh = [&](float pm, float pl) {
            const float mn = fmaxf(M, warp_max(pl != 0.f ? pm : -INFINITY)), mu = mn == -INFINITY ? 0.f : mn, c = pt_ex2(M - mu), e = pl != 0.f ? pt_ex2(pm - mu) : 0.f;
            L = fmaf(L, c, warp_sum(pl * e));
            O = make_float4(O.x * c, O.y * c, O.z * c, O.w * c);
            M = mn;
            return e;
        };
        {
            const bool mine = lane < WARPS;
            const float e = weigh(mine ? w_ml[(lane * G + h) * 2] : -INFINITY, mine ? w_ml[(lane * G + h) * 2 + 1] : 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float ew = __shfl_sync(0xffffffffu, e, w);
                if (half == 0 && ew != 0.f) put(*reinterpret_cast<const float4*>(w_acc + (w * G + h) * HS + d4 * 4), ew);
            }
        }
        if (shared > 0) {
            const int r = (m - plan.begin[g_of]) * G + h, t = r / SH_ROWS;
            ShUnit unit;
            sh_unit(a, plan, g_of, kvh, t / 2, unit);
            const int b0 = sh_quot(unit.c0, plan.quota) + rank, b1 = sh_quot(unit.c0 + unit.steps * unit.w - 1, plan.quota) + 1, n = b1 > b0 ? (b1 - b0 + n_cl - 1) / n_cl : 0;
            const float2* norms = sh_norms(a) + r % SH_ROWS;
            const float4* sums = sh_sums(a) + r % SH_ROWS * LPH + d4;
            for (int c0 = 0; c0 < n; c0 += 32) {
                const int c = c0 + lane, b = b0 + c * n_cl;
                int j0 = 0, j1 = 0;
                if (c < n) sh_share(plan, unit, b, j0, j1);
                const unsigned at = (unsigned)(unit.index + b) * 2 + (t & 1);
                const bool there = j1 > j0;
                const unsigned all = __ballot_sync(0xffffffffu, there);
                const float2 x = there ? __ldcg(norms + (size_t)at * SH_ROWS) : make_float2(-INFINITY, 0.f);
                const int live = min(32, n - c0);
                constexpr int BY = 32 / LPH, FLY = 16;           // pieces a load, loads in flight: the first ones together with the norms
                float4 v[FLY];
                auto fetch = [&](int i0) {
#pragma unroll
                    for (int i = 0; i < FLY; i++) {
                        const int from = (i0 + i * BY + half) & 31;
                        const unsigned where = __shfl_sync(0xffffffffu, at, from);
                        v[i] = all >> from & 1 && i0 + i * BY < live ? __ldcg(sums + (size_t)where * SH_ROWS * LPH) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                };
                fetch(0);
                const float e = weigh(x.x, x.y);
#pragma unroll 1
                for (int i0 = 0; i0 < live; i0 += FLY * BY) {
                    if (i0 > 0) fetch(i0);
#pragma unroll
                    for (int i = 0; i < FLY; i++) {
                        const int from = i0 + i * BY + half;
                        const float f = __shfl_sync(0xffffffffu, e, from & 31);
                        if (from < live && f != 0.f) put(v[i], f);      // (a piece in which nothing was seen may hold anything)
                    }
                }
            }
        }
        if (HS == 64) {
            O.x += __shfl_xor_sync(0xffffffffu, O.x, 16); O.y += __shfl_xor_sync(0xffffffffu, O.y, 16);
            O.z += __shfl_xor_sync(0xffffffffu, O.z, 16); O.w += __shfl_xor_sync(0xffffffffu, O.w, 16);
        }
        if (half == 0) *reinterpret_cast<float4*>(c_acc + h * HS + d4 * 4) = O;
        if (lane == 0) { c_ml[h * 2] = M; c_ml[h * 2 + 1] = bad_s ? __int_as_float(0x7fffffff) : L; }
    }
    if (n_cl > 1) cluster.sync();
    else __syncthreads();
    // blocks of 32 values, a warp each: over the CTAs of the cluster
    for (int blk = rank * WARPS + warp; blk < G * (HS / 32); blk += n_cl * WARPS) {
        const int h = blk / (HS / 32), d = blk % (HS / 32) * 32 + lane;
        float M = -INFINITY, L = 0.f, O = 0.f;
        for (int r = 0; r < n_cl; r++) {
            const float* ml = n_cl > 1 ? cluster.map_shared_rank(c_ml, r) : c_ml;
            const float* acc = n_cl > 1 ? cluster.map_shared_rank(c_acc, r) : c_acc;
            const float pm = ml[h * 2], pl = ml[h * 2 + 1], x = acc[h * HS + d];
            if (pl == 0.f) continue;
            const float mn = fmaxf(M, pm), mu = mn == -INFINITY ? 0.f : mn, c = pt_ex2(M - mu), e = pt_ex2(pm - mu);
            L = fmaf(L, c, pl * e);
            O = fmaf(O, c, x * e);
            M = mn;
        }
        float y = O / L;
        if (T == 0) y = 0.f;                                     // no token
        else if (T < 0 || !(L > 0.f)) y = __int_as_float(0x7fffffff);
        const int col = (kvh * G + h) * HS + d;
        if (a.y_out != nullptr) {
            const size_t at = (size_t)((long long)m * a.ldy + col);
            if (a.y_type == DL_KV8_F32) reinterpret_cast<float*>(a.y_out)[at] = y;
            else if (a.y_type == DL_KV8_BF16) reinterpret_cast<__nv_bfloat16*>(a.y_out)[at] = __float2bfloat16(y);
            else reinterpret_cast<__half*>(a.y_out)[at] = __float2half_rn(y);
        }
        if (a.xq_out != nullptr || a.xh_out != nullptr) q80_block_store(y, lane, m, col >> 5, a.out_mcap, a.xq_out, a.xh_out);
    }
    if (n_cl > 1) cluster.sync();                                // nobody leaves while its sums are read
}

#define SH_SMEM ((2 + 2 * SH_STAGES) * SH_TILE_BYTES + 8 * 32 * SH_OUT_LD * 4 + 20 * 8)

static size_t sh_own_smem(int head_size, int G, int warps) {
    const size_t ring = (size_t)warps * (256 / head_size) * 2 * SH_OWN_TOK * head_size * 2;
    const size_t join = (size_t)(warps + 1) * G * (head_size + 2) * 4;
    return ring > join ? ring : join;
}

// pieces at most: a unit more with every share that begins in it
static long long sh_pieces(long long M, int n_heads, int n_kv_heads) {
    const long long rep = n_heads / n_kv_heads;
    return n_kv_heads * (M * rep / (2 * SH_ROWS) + SH_MAX_GROUPS + 1) + dl_device_sm_count();
}

extern "C" long long dl_shared_attention_scratch_bytes(int M, int n_heads, int n_kv_heads, int head_size) {
    if (M < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 || head_size < 1) return 0;
    return sh_pieces(M, n_heads, n_kv_heads) * 2 * SH_ROWS * (8 + (long long)head_size * 4);
}

static int sh_map(CUtensorMap* map, const void* base, long long rows, int width) {
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)width * 2};
    const cuuint32_t box[2] = {64, SH_PAGE};
    return dl_tensor_map("dl_shared_attention", map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int HS> static int sh_launch(const ShArgs& a, int pdl, cudaStream_t stream) {
    alignas(64) CUtensorMap kmap, vmap;
    const long long rows = (long long)a.n_pages * a.n_kv_heads * SH_PAGE;
    if (sh_map(&kmap, a.k_cache, rows, HS) != 0 || sh_map(&vmap, a.v_cache, rows, HS) != 0) return -1;
    WaitLimit limit;
    if (dl_wait_limit("dl_shared_attention", &limit) != 0) return -1;
    const int G = a.n_heads / a.n_kv_heads, n_sms = dl_device_sm_count();
    // Many rows: two warps for each, so that an SM has six of them at work: what bounds a row are its latencies, one behind the other
    const bool many = (long long)a.M * a.n_kv_heads > 3ll * n_sms;
    const int warps = many ? 2 : 4;
    // (rows 8 to 15 of the MMAs and what belongs to them only where there are so many heads)
    auto* own_kernel = G > 8 ? (many ? shared_own_kernel<HS, 2, 2> : shared_own_kernel<HS, 4, 2>) : many ? shared_own_kernel<HS, 2, 1> : shared_own_kernel<HS, 4, 1>;
    static SmemLimit given, given_own[2][2];
    const size_t own_smem = sh_own_smem(HS, G, warps);
    if (const int rc = dl_smem_limit("dl_shared_attention", shared_attention_kernel<HS>, SH_SMEM, given)) return rc;
    if (const int rc = dl_smem_limit("dl_shared_attention", own_kernel, own_smem, given_own[many][G > 8])) return rc;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    cfg.gridDim = dim3(a.shares);
    cfg.blockDim = dim3(SH_THREADS);
    cfg.dynamicSmemBytes = SH_SMEM;
    cfg.stream = stream;
    cudaError_t e = cudaLaunchKernelEx(&cfg, shared_attention_kernel<HS>, a, kmap, vmap, limit);
    if (e == cudaSuccess) {
        // few rows: a cluster for each row and key/value head
        int ctas = 1;
        while (ctas < SH_OWN_MAX_CTAS && (long long)a.M * a.n_kv_heads * ctas * 2 <= 2ll * n_sms) ctas *= 2;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = ctas;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
        cfg.gridDim = dim3(ctas, a.n_kv_heads, a.M);
        cfg.blockDim = dim3(warps * 32);
        cfg.dynamicSmemBytes = own_smem;
        e = cudaLaunchKernelEx(&cfg, own_kernel, a);
    }
    if (e != cudaSuccess) { dl_set_error("dl_shared_attention launch: %s", cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

extern "C" int dl_shared_attention(const float* q, long long ldq, int n_heads, int n_kv_heads, int head_size, const void* k_cache, const void* v_cache, int n_pages, const int* pos, const int* slot,
                                   const int* block_table, int M, int n_slots, int max_pages, const int* groups, int max_groups, void* scratch, long long scratch_bytes, uint8_t* xq_out,
                                   uint8_t* xh_out, int out_mcap, void* y_out, long long ldy, int y_type, int pdl, void* stream) {
    if (head_size != 64 && head_size != 128) { dl_set_error("dl_shared_attention: heads of 64 and 128, not %d", head_size); return -1; }
    if (n_kv_heads < 1 || n_kv_heads > 65535 || n_heads < 1 || n_heads % n_kv_heads != 0 || n_heads / n_kv_heads > 16) { dl_set_error("dl_shared_attention: unsupported head grouping %d/%d", n_heads, n_kv_heads); return -1; }
    if (M < 0 || M > 65535 || n_slots < 1 || max_pages < 1 || max_pages > 1 << 25 || n_pages < 1 || max_groups < 0 || (long long)n_pages * n_kv_heads * SH_PAGE > 0x7fffffffll) {
        dl_set_error("dl_shared_attention: %d rows, %d tables of %d pages, %d pages, %d groups", M, n_slots, max_pages, n_pages, max_groups);
        return -1;
    }
    if (M == 0) return 0;
    if (!q || !k_cache || !v_cache || !pos || !slot || !block_table || !groups || !scratch) { dl_set_error("dl_shared_attention: a null pointer"); return -1; }
    if (scratch_bytes < dl_shared_attention_scratch_bytes(M, n_heads, n_kv_heads, head_size)) { dl_set_error("dl_shared_attention: a scratch of %lld bytes is too small", scratch_bytes); return -1; }
    if (n_kv_heads * ((long long)M * (n_heads / n_kv_heads) / (2 * SH_ROWS) + SH_MAX_GROUPS + 1) * SH_PAIR_COST * (max_pages / (SH_KV / SH_PAGE) + 1) > 1ll << 30) {
        dl_set_error("dl_shared_attention: %d rows with tables of %d pages are too much for one launch", M, max_pages);
        return -1;
    }
    const long long cols = (long long)n_heads * head_size;
    if (ldq < cols || ldq % 4 != 0 || (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)scratch) & 15) != 0) { dl_set_error("dl_shared_attention: q, cache and scratch are aligned to 16 bytes, rows of q to 4 values"); return -1; }
    if (y_out != nullptr && (ldy < cols || (y_type != DL_KV8_F32 && y_type != DL_KV8_BF16 && y_type != DL_KV8_F16))) { dl_set_error("dl_shared_attention: y_out of type %d, row stride %lld", y_type, ldy); return -1; }
    const ShArgs a = {q, ldq, (const __half*)k_cache, (const __half*)v_cache, pos, slot, block_table, groups, M, n_heads, n_kv_heads, n_heads / n_kv_heads, n_slots, max_pages, n_pages, max_groups,
                      (uint8_t*)scratch, dl_device_sm_count(), sh_pieces(M, n_heads, n_kv_heads), xq_out, xh_out, out_mcap, y_out, ldy, y_type};
    return head_size == 128 ? sh_launch<128>(a, pdl, (cudaStream_t)stream) : sh_launch<64>(a, pdl, (cudaStream_t)stream);
}
