// Block tables and slot maps from the requests' lengths, so that a loop of steps takes the pages it needs without the host.
//
// Request i of n holds held[i] tokens in the pages of table row seq[i] and runs new[i] more:
//   have = ceil(held / 32), need = ceil((held + new) / 32) pages; P and R: sums of need - have and of new over the requests ahead
//   table[seq][k] = free[taken + P + k - have], have <= k < need;  table[seq][k] = table[lead_seq][k], k < lead_pages (a shared prompt)
//   pos[R + j] = held + j, slot[R + j] = seq, line[R + j] = 32 table[seq][pos / 32] + pos % 32; rows behind the last one: -1, 0, -1
// All of it happens or nothing: every CTA checks everything by itself (lengths are a few KB), and where something is wrong `status` says what, all
// rows are left empty and nothing is taken.
//
// What bounds it: the chain of latencies (lengths, sums, free pages, table, rows), and for many requests the shared pages' copies.  So every CTA forms all sums, for which a barrier in between would cost
// more, and writes its part of the results; a row finds its request by bisection over the sums in shared memory.  Where lengths and the count of taken pages are updated in place, one cluster does
// it all: its CTAs have all read before one writes.  32 requests of a token each 5.2 us, 2001 requests with 22000 rows behind 250 shared pages 11.6 (27.8 by one cluster).
#include "../../../include/dllama_b200.h"
#include "common.cuh"
#include "smem_limit.cuh"

#define PGT_THREADS 1024
#define PGT_PAGE 32
#define PGT_MAX_REQUESTS 8192
#define PGT_MAX_SEQS 131072
#define PGT_MAX_CLUSTERS 8
#define PGT_UNIT 128                   // shared pages that a warp copies at a time

extern void dl_set_error(const char* fmt, ...);


struct PgtArgs {
    const int *held, *new_tokens, *seq, *lead_seq, *lead_pages;
    int* table;
    const int *free_pages, *taken;
    int *pos, *slot, *line, *start, *held_out, *taken_out, *status;
    int n, n_seqs, max_pages, n_free, n_pages, M;
};

// the last i with at[i] <= x (at[0] = 0, x < at[n])
DL_DEVINL int pgt_find(const uint32_t* at, int n, uint32_t x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PGT_THREADS) page_tables_kernel(const __grid_constant__ PgtArgs a) {
    extern __shared__ uint32_t sm[];
    __shared__ unsigned long long warp_sums[3][32];
    const int n = a.n, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cta = blockIdx.x, ctas = gridDim.x;              // (one cluster where results go in place)
    const int words = (a.n_seqs + 31) / 32;
    uint32_t* row_at = sm;                                     // [n + 1] rows, pages and units of shared pages ahead of a request
    uint32_t* page_at = row_at + n + 1;
    uint32_t* unit_at = page_at + n + 1;
    int* held = reinterpret_cast<int*>(unit_at + n + 1);       // [n]
    int* seq = held + n;                                       // [n]
    uint32_t* used = reinterpret_cast<uint32_t*>(seq + n);     // [words] table rows of requests
    uint32_t* led = used + words;                              // [words] ... whose first pages are another's
    uint32_t* grown = led + words;                             // [words] ... that get pages in this call
    pdl_launch_dependents();
    for (int i = tid; i < 3 * words; i += PGT_THREADS) used[i] = 0;
    __syncthreads();
    pdl_wait();
    const int taken = *a.taken;
    const int per = (n + PGT_THREADS - 1) / PGT_THREADS, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const bool leads = a.lead_seq != nullptr;
    int bad = 0;
    unsigned long long sum[3] = {0, 0, 0};
    for (int i = i0; i < i1; i++) {
        const int h = a.held[i], c = a.new_tokens[i], s = a.seq[i], l = leads ? a.lead_pages[i] : 0;
        held[i] = h;
        seq[i] = s;
        if (h < 0 || c < 0 || (long long)h + c > (long long)a.max_pages * PGT_PAGE) { bad |= DL_TABLES_BAD_LENGTH; continue; }
        const bool lead_ok = l >= 0 && (long long)l * PGT_PAGE <= h && (l == 0 || (unsigned)a.lead_seq[i] < (unsigned)a.n_seqs);
        const int more = (h + c + PGT_PAGE - 1) / PGT_PAGE - (h + PGT_PAGE - 1) / PGT_PAGE;
        if (!lead_ok) bad |= DL_TABLES_BAD_LEAD;
        if ((unsigned)s >= (unsigned)a.n_seqs) bad |= DL_TABLES_BAD_SEQ;
        else {
            if (atomicOr(&used[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) bad |= DL_TABLES_BAD_SEQ;
            if (lead_ok && l > 0 && a.lead_seq[i] != s) atomicOr(&led[s >> 5], 1u << (s & 31));
            if (leads && more > 0) atomicOr(&grown[s >> 5], 1u << (s & 31));
        }
        sum[0] += c;
        sum[1] += more;
        sum[2] += lead_ok ? (l + PGT_UNIT - 1) / PGT_UNIT : 0;
    }
    unsigned long long incl[3];
#pragma unroll
    for (int q = 0; q < 3; q++) {
        incl[q] = sum[q];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long x = __shfl_up_sync(0xffffffffu, incl[q], o);
            if (lane >= o) incl[q] += x;
        }
        if (lane == 31) warp_sums[q][warp] = incl[q];
    }
    __syncthreads();
    unsigned long long ahead[3], total[3];
#pragma unroll
    for (int q = 0; q < 3; q++) {
        unsigned long long x = warp_sums[q][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        total[q] = __shfl_sync(0xffffffffu, x, 31);
        const unsigned long long before = __shfl_sync(0xffffffffu, x, max(warp - 1, 0));
        ahead[q] = (warp ? before : 0) + incl[q] - sum[q];
    }
    int grown_lead = -1, grown_have = 0;                       // a table row that gets pages in this call, and how many it has
    for (int i = i0; i < i1; i++) {
        row_at[i] = (uint32_t)ahead[0];
        page_at[i] = (uint32_t)ahead[1];
        unit_at[i] = (uint32_t)ahead[2];
        const int h = held[i], c = a.new_tokens[i], l = leads ? a.lead_pages[i] : 0;
        ahead[0] += c;
        ahead[1] += ((long long)h + c + PGT_PAGE - 1) / PGT_PAGE - ((long long)h + PGT_PAGE - 1) / PGT_PAGE;
        ahead[2] += l > 0 ? (l + PGT_UNIT - 1) / PGT_UNIT : 0;
        if (l > 0 && bad == 0) {                   // pages of a row that gets its own from another in this call, or that this call takes for it
            const int t = a.lead_seq[i];
            if (t != seq[i] && (led[t >> 5] >> (t & 31) & 1)) bad |= DL_TABLES_BAD_LEAD;
            if (t != seq[i] && (grown[t >> 5] >> (t & 31) & 1)) {
                if (t != grown_lead)               // (seldom: whose request it is, nobody has noted)
                    for (int j = 0; j < n; j++)
                        if (seq[j] == t) { grown_lead = t; grown_have = (held[j] + PGT_PAGE - 1) / PGT_PAGE; }
                if (l > grown_have) bad |= DL_TABLES_BAD_LEAD;
            }
        }
    }
    if (tid == 0) {
        row_at[n] = (uint32_t)total[0];
        page_at[n] = (uint32_t)total[1];
        unit_at[n] = (uint32_t)total[2];
        if (total[0] > (unsigned long long)a.M) bad |= DL_TABLES_NO_ROWS;
        if (taken < 0 || (unsigned long long)taken + total[1] > (unsigned long long)a.n_free) bad |= DL_TABLES_NO_PAGES;
    }
    if (taken >= 0 && total[1] <= (unsigned long long)a.n_free && (unsigned long long)taken + total[1] <= (unsigned long long)a.n_free)
        for (int j = tid; j < (int)total[1]; j += PGT_THREADS)
            if ((unsigned)a.free_pages[taken + j] >= (unsigned)a.n_pages) bad |= DL_TABLES_BAD_PAGE;
#pragma unroll
    for (int b = 1; b <= DL_TABLES_NO_ROWS; b <<= 1) if (__syncthreads_or(bad & b)) bad |= b;
    // every CTA has read what one of them may write
    if (ctas > 1) { cg::this_cluster().sync(); }
    const int n_rows = bad ? 0 : (int)total[0], n_new = bad ? 0 : (int)total[1], n_units = bad ? 0 : (int)total[2];
    const int t0 = cta * PGT_THREADS + tid, step = ctas * PGT_THREADS;
    for (int r = t0; r < a.M; r += step) {
        int p = -1, s = 0, line = -1;
        if (r < n_rows) {
            const int i = pgt_find(row_at, n, r), have = (held[i] + PGT_PAGE - 1) / PGT_PAGE;
            p = held[i] + (r - (int)row_at[i]);
            s = seq[i];
            if (a.line != nullptr) {
                const int k = p / PGT_PAGE, page = k >= have ? a.free_pages[taken + (int)page_at[i] + k - have] : a.table[(size_t)s * a.max_pages + k];
                if ((unsigned)page < (unsigned)a.n_pages) line = page * PGT_PAGE + p % PGT_PAGE;
            }
        }
        a.pos[r] = p;
        a.slot[r] = s;
        if (a.line != nullptr) a.line[r] = line;
    }
    for (int j = t0; j < n_new; j += step) {
        const int i = pgt_find(page_at, n, j), k = (held[i] + PGT_PAGE - 1) / PGT_PAGE + (j - (int)page_at[i]);
        a.table[(size_t)seq[i] * a.max_pages + k] = a.free_pages[taken + j];
    }
    for (int u = t0 >> 5; u < n_units; u += step >> 5) {
        const int i = pgt_find(unit_at, n, u), k0 = (u - (int)unit_at[i]) * PGT_UNIT, l = a.lead_pages[i];
        const int* src = a.table + (size_t)a.lead_seq[i] * a.max_pages;
        int* dst = a.table + (size_t)seq[i] * a.max_pages;
        int v[PGT_UNIT / 32];
#pragma unroll
        for (int q = 0; q < PGT_UNIT / 32; q++) if (k0 + q * 32 + lane < l) v[q] = src[k0 + q * 32 + lane];
#pragma unroll
        for (int q = 0; q < PGT_UNIT / 32; q++) if (k0 + q * 32 + lane < l) dst[k0 + q * 32 + lane] = v[q];
    }
    for (int i = t0; i < n; i += step) a.held_out[i] = held[i] + (bad ? 0 : (int)(row_at[i + 1] - row_at[i]));
    if (a.start != nullptr)
        for (int i = t0; i <= n; i += step) a.start[i] = bad ? 0 : (int)row_at[i];
    if (t0 == 0) {
        *a.taken_out = taken + n_new;
        *a.status = bad;
    }
}

extern "C" int dl_page_tables(int n, const int* held, const int* new_tokens, const int* seq, int* table, int n_seqs, int max_pages, const int* free_pages, int n_free, const int* taken,
                              int n_pages, int M, int* pos, int* slot, int* line, int* start, int* held_out, int* taken_out, int* status, const int* lead_seq, const int* lead_pages, int pdl,
                              void* stream) {
    if (n < 0 || n > PGT_MAX_REQUESTS || n_seqs < 1 || n_seqs > PGT_MAX_SEQS) { dl_set_error("dl_page_tables: %d requests (at most %d), %d table rows (1 to %d)", n, PGT_MAX_REQUESTS, n_seqs, PGT_MAX_SEQS); return -1; }
    if (max_pages < 1 || max_pages > 1 << 25 || n_free < 0 || n_free > 1 << 30 || n_pages < 1 || n_pages > 1 << 26 || M < 0 || M > 1 << 30) { dl_set_error("dl_page_tables: tables of %d pages, %d free of %d pages, %d rows", max_pages, n_free, n_pages, M); return -1; }
    if (!table || !taken || !taken_out || !status || (n > 0 && (!held || !new_tokens || !seq || !held_out)) || (n_free > 0 && !free_pages) || (M > 0 && (!pos || !slot)) || !lead_seq != !lead_pages) {
        dl_set_error("dl_page_tables: a null pointer");
        return -1;
    }
    const PgtArgs a = {held, new_tokens, seq, lead_seq, lead_pages, table, free_pages, taken, pos, slot, line, start, held_out, taken_out, status, n, n_seqs, max_pages, n_free, n_pages, M};
    const size_t smem = ((size_t)3 * (n + 1) + 2 * (size_t)n + 3 * (size_t)((n_seqs + 31) / 32)) * 4;
    static SmemLimit given;
    if (smem > 48 * 1024)
        if (const int rc = dl_smem_limit("dl_page_tables", page_tables_kernel, smem, given)) return rc;
    // one CTA where a barrier among several would cost more than their stores gain; clusters of eight for every 8192 rows (and requests with shared pages, each as so many) up to half of the SMs
    const long long work = (long long)M + (lead_seq ? 64ll * n : 0);
    const int ctas = work <= 2048 ? 1 : work <= 4096 ? 2 : work <= 8192 ? 4 : 8;
    const bool in_place = (held_out < held + n && held < held_out + n) || taken_out == taken;
    const int clusters = in_place || work <= 8192 ? 1 : (int)(work / 8192 < PGT_MAX_CLUSTERS ? work / 8192 : PGT_MAX_CLUSTERS);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas * clusters);
    cfg.blockDim = dim3(PGT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, page_tables_kernel, a);
    if (e != cudaSuccess) { dl_set_error("dl_page_tables launch: %s", cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

extern "C" int dl_page_tables_packed(const DlPageTables* a) {
    if (!a) { dl_set_error("dl_page_tables: a null pointer"); return -1; }
    const long long counts[] = {a->n, a->n_seqs, a->max_pages, a->n_free, a->n_pages, a->M};
    for (long long c : counts)
        if (c != (int)c) { dl_set_error("dl_page_tables: a count of %lld", c); return -1; }
    return dl_page_tables((int)a->n, a->held, a->new_tokens, a->seq, a->table, (int)a->n_seqs, (int)a->max_pages, a->free_pages, (int)a->n_free, a->taken, (int)a->n_pages, (int)a->M, a->pos, a->slot, a->line,
                          a->start, a->held_out, a->taken_out, a->status, a->lead_seq, a->lead_pages, a->pdl != 0, a->stream);
}
