// Paged grouped-query attention over the 8-bit token cache (kv8.cuh has the format): decode rows and prompt chunks.
//
// Reference semantics: OP_MULTIHEAD_ATT (multiheadAtt_F32, src/nn/nn-cpu-ops.cpp:749-784) over the positions 0..pos of each row, softmax in f32, with
// keys and values as the cache holds them; output f32 (or rounded once to 16 bits) and / or cast to Q80 in the slabs that the wo matmul consumes
// (OP_CAST, src/llm.cpp:296-301).
//
// A row without tokens (a negative position) gives zeros; one whose sequence, position or page is not in the tables, or whose query is not finite,
// gives NaN, and so does a token whose line holds a NaN to the rows that see it.
#include <math.h>
#include <type_traits>
#include "epilogue.cuh"
#include "kv8.cuh"

extern void dl_set_error(const char* fmt, ...);
extern int kv8_check(const char* who, const DlKv8Cache* c, const DlKv8Rows* r);

struct Kv8AttArgs {
    const float* q;            // [M][ldq]
    long long ldq;
    Kv8Rows rows;
    DlKv8Cache c;
    int heads;
    const int* row_skip;       // NULL, or row_skip[m] != 0: not this launch's row
    const int* meta;           // NULL, or rows outside its segments are not this launch's
    uint8_t* xq_out;
    uint8_t* xh_out;
    int out_mcap;
    void* y_out;               // [M][ldy] or NULL
    long long ldy;
    int y_type;
};

DL_DEVINL void kv8_store_y(const Kv8AttArgs& a, int m, int col, float y) {
    if (a.y_out == nullptr) return;
    const size_t at = (size_t)m * a.ldy + col;
    if (a.y_type == DL_KV8_F32) reinterpret_cast<float*>(a.y_out)[at] = y;
    else if (a.y_type == DL_KV8_BF16) reinterpret_cast<__nv_bfloat16*>(a.y_out)[at] = __float2bfloat16_rn(y);
    else reinterpret_cast<__half*>(a.y_out)[at] = __float2half_rn(y);
}

// a warp per row and head, lane = head dimension of each block of 32
template <int HS>
__global__ void __launch_bounds__(128) kv8_attention_rows_kernel(const __grid_constant__ Kv8AttArgs a) {
    constexpr int DPL = HS / 32;
    const int lane = threadIdx.x & 31, m = blockIdx.y, head = blockIdx.x * 4 + (threadIdx.x >> 5);
    pdl_launch_dependents();
    pdl_wait();
    if (head >= a.heads || (a.row_skip != nullptr && a.row_skip[m] != 0)) return;
    if (a.meta != nullptr) {
        bool mine = false;
        for (int i = 0; i < min(a.meta[0], 8); i++) mine |= m >= a.meta[1 + 2 * i] && m < a.meta[2 + 2 * i];
        if (!mine) return;
    }
    const int kvh = head / (a.heads / a.c.n_kv_heads), slot = a.rows.slot[m];
    int T = kv8_tokens(a.rows, a.rows.pos[m], slot);
    bool bad = T < 0;
    float q[DPL], o[DPL], mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DPL; d++) { q[d] = a.q[m * a.ldq + head * HS + d * 32 + lane] * rsqrtf((float)HS); o[d] = 0.f; }
    for (int t = 0; t < T; t++) {
        const int page = a.rows.block_table[(size_t)slot * a.rows.max_pages + t / KV8_PAGE];
        if ((unsigned)page >= (unsigned)a.rows.n_pages) { bad = true; break; }
        const size_t line = ((size_t)page * a.c.n_kv_heads + kvh) * KV8_PAGE + t % KV8_PAGE;
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < DPL; d++) s = fmaf(q[d], (float)a.c.k[line * HS + d * 32 + lane], s);
        s = warp_sum(s) * a.c.k_scale[line];
        const float mn = fmaxf(mx, s), mu = mn == -INFINITY ? 0.f : mn, corr = __expf(mx - mu), p = __expf(s - mu), pv = p * a.c.v_scale[line];
        mx = mn;
        l = fmaf(l, corr, p);
#pragma unroll
        for (int d = 0; d < DPL; d++) o[d] = fmaf(o[d], corr, pv * (float)a.c.v[line * HS + d * 32 + lane]);
    }
#pragma unroll
    for (int d = 0; d < DPL; d++) {
        const float y = bad ? __uint_as_float(0x7fffffffu) : l == 0.f ? 0.f : o[d] / l;
        kv8_store_y(a, m, head * HS + d * 32 + lane, y);
        if (a.xq_out != nullptr || a.xh_out != nullptr) q80_block_store(y, lane, m, head * DPL + d, a.out_mcap, a.xq_out, a.xh_out);
    }
}

static int kv8_rows_launch(const char* who, const Kv8AttArgs& a, int pdl, void* stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.heads + 3) / 4, a.rows.M);
    cfg.blockDim = dim3(128);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    if (pdl) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    const int hs = a.c.head_size;
    const cudaError_t e = hs == 128 ? cudaLaunchKernelEx(&cfg, kv8_attention_rows_kernel<128>, a)
                          : hs == 64 ? cudaLaunchKernelEx(&cfg, kv8_attention_rows_kernel<64>, a)
                                     : cudaLaunchKernelEx(&cfg, kv8_attention_rows_kernel<32>, a);
    if (e != cudaSuccess) { dl_set_error("%s launch: %s", who, cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

// what both entry points refuse
static int kv8_att_args(const char* who, const float* q, long long ldq, int n_heads, const DlKv8Rows* rows, const DlKv8Cache* cache, uint8_t* xq_out, uint8_t* xh_out,
                        int out_mcap, void* y_out, long long ldy, int y_type, Kv8AttArgs* a) {
    if (const int rc = kv8_check(who, cache, rows)) return rc;
    const int hs = cache->head_size, kv = cache->n_kv_heads;
    if (n_heads < kv || n_heads % kv != 0 || n_heads / kv > 16) { dl_set_error("%s: unsupported head grouping %d/%d", who, n_heads, kv); return -1; }
    if (q == nullptr || (xq_out == nullptr && xh_out == nullptr && y_out == nullptr)) { dl_set_error("%s: no queries or no output", who); return -1; }
    if (ldq < (long long)n_heads * hs || (y_out != nullptr && ldy < (long long)n_heads * hs)) { dl_set_error("%s: rows overlap (ld %lld, %lld)", who, ldq, ldy); return -1; }
    if (y_type != DL_KV8_F32 && y_type != DL_KV8_BF16 && y_type != DL_KV8_F16) { dl_set_error("%s: unsupported output type %d", who, y_type); return -1; }
    if ((xq_out != nullptr || xh_out != nullptr) && ((long long)n_heads * hs % 128 != 0 || out_mcap < rows->M || (xh_out != nullptr && out_mcap % 8 != 0))) {
        dl_set_error("%s: slabs of %d rows, %d columns", who, out_mcap, n_heads * hs);
        return -1;
    }
    *a = {q, ldq, {rows->pos, rows->slot, rows->block_table, rows->M, rows->n_slots, rows->max_pages, cache->n_pages}, *cache, n_heads, nullptr, nullptr, xq_out, xh_out, out_mcap, y_out, ldy, y_type};
    if (rows->M > 65535) { dl_set_error("%s: %d rows (65535 at most)", who, rows->M); return -1; }
    return 0;
}

extern "C" int dl_kv8_attention(const float* q, long long ldq, int n_heads, const DlKv8Rows* rows, const DlKv8Cache* cache, int n_splits, void* scratch, uint8_t* xq_out,
                                uint8_t* xh_out, int out_mcap, void* y_out, long long ldy, int y_type, const int* row_skip, int pdl, void* stream) {
    Kv8AttArgs a;
    if (const int rc = kv8_att_args("dl_kv8_attention", q, ldq, n_heads, rows, cache, xq_out, xh_out, out_mcap, y_out, ldy, y_type, &a)) return rc;
    if (n_splits > 1 && scratch == nullptr) { dl_set_error("dl_kv8_attention: n_splits>1 needs scratch"); return -1; }
    if (rows->M == 0) return 0;
    a.row_skip = row_skip;
    return kv8_rows_launch("dl_kv8_attention", a, pdl, stream);
}

extern "C" int dl_kv8_attention_prefill(const float* q, long long ldq, int n_heads, const DlKv8Rows* rows, const int* meta, const DlKv8Cache* cache, void* k16, void* v16,
                                        uint8_t* xq_out, uint8_t* xh_out, int out_mcap, void* y_out, long long ldy, int y_type, int pdl, void* stream) {
    Kv8AttArgs a;
    if (const int rc = kv8_att_args("dl_kv8_attention_prefill", q, ldq, n_heads, rows, cache, xq_out, xh_out, out_mcap, y_out, ldy, y_type, &a)) return rc;
    if (meta == nullptr || (k16 == nullptr) != (v16 == nullptr)) { dl_set_error("dl_kv8_attention_prefill: a null pointer"); return -1; }
    if (rows->M == 0) return 0;
    a.meta = meta;
    return kv8_rows_launch("dl_kv8_attention_prefill", a, pdl, stream);
}
