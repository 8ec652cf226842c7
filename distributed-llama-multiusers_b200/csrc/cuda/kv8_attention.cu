// Paged grouped-query attention over the 8-bit token cache (kv8.cuh has the format): decode rows and prompt chunks.
//
// Reference semantics: OP_MULTIHEAD_ATT (multiheadAtt_F32, src/nn/nn-cpu-ops.cpp:749-784) over the positions 0..pos of each row, softmax in f32, with
// keys and values as the cache holds them; output f32 (or rounded once to 16 bits) and / or cast to Q80 in the slabs that the wo matmul consumes
// (OP_CAST, src/llm.cpp:296-301).
//
// A row without tokens (a negative position) gives zeros; one whose sequence, position or page is not in the tables, whose query is not finite or whose
// scores are all below what f32 holds gives NaN, and so does a token whose line holds a NaN to the rows that see it.
#include <math.h>
#include <type_traits>
#include "epilogue.cuh"
#include "kv8.cuh"
#include "prefill_shares.cuh"
#include "smem_limit.cuh"

extern void dl_set_error(const char* fmt, ...);
extern int dl_device_sm_count();
extern int kv8_check(const char* who, const DlKv8Cache* c, const Kv8Rows* r);

struct Kv8AttArgs {
    const float* q;            // [M][ldq]
    long long ldq;
    Kv8Rows rows;
    DlKv8Cache c;
    int heads;
    const int* row_skip;       // NULL, or row_skip[m] != 0: not this launch's row
    const int* meta;           // NULL, or rows outside its segments are not this launch's
    int n_seg;                 // segments that are looked at, at most
    uint8_t* xq_out;
    uint8_t* xh_out;
    int out_mcap;
    void* y_out;               // [M][ldy] or NULL
    long long ldy;
    int y_type;
    bool y_vec;                // rows of y_out take four values at once
};

DL_DEVINL void kv8_store_y(const Kv8AttArgs& a, int m, int col, float y) {
    if (a.y_out == nullptr) return;
    const size_t at = (size_t)m * a.ldy + col;
    if (a.y_type == DL_KV8_F32) reinterpret_cast<float*>(a.y_out)[at] = y;
    else if (a.y_type == DL_KV8_BF16) reinterpret_cast<__nv_bfloat16*>(a.y_out)[at] = __float2bfloat16_rn(y);
    else reinterpret_cast<__half*>(a.y_out)[at] = __float2half_rn(y);
}

// four neighbouring values of a row from column col on, eight lanes side by side a Q80 block of 32 (by whole warps; live: the lane has any)
DL_DEVINL void kv8_store4(const Kv8AttArgs& a, int m, int col, float4 y, bool live, int lane) {
    if (a.y_out != nullptr && live) {
        const size_t at = (size_t)m * a.ldy + col;
        if (a.y_type == DL_KV8_F32) {
            float* d = reinterpret_cast<float*>(a.y_out) + at;
            if (a.y_vec) *reinterpret_cast<float4*>(d) = y;
            else { d[0] = y.x; d[1] = y.y; d[2] = y.z; d[3] = y.w; }
        } else {
            uint32_t lo, hi;
            if (a.y_type == DL_KV8_BF16) {
                const __nv_bfloat162 u = __floats2bfloat162_rn(y.x, y.y), v = __floats2bfloat162_rn(y.z, y.w);
                lo = *reinterpret_cast<const uint32_t*>(&u);
                hi = *reinterpret_cast<const uint32_t*>(&v);
            } else {
                const __half2 u = __floats2half2_rn(y.x, y.y), v = __floats2half2_rn(y.z, y.w);
                lo = *reinterpret_cast<const uint32_t*>(&u);
                hi = *reinterpret_cast<const uint32_t*>(&v);
            }
            uint16_t* d = reinterpret_cast<uint16_t*>(a.y_out) + at;
            if (a.y_vec) *reinterpret_cast<uint2*>(d) = make_uint2(lo, hi);
            else { d[0] = (uint16_t)lo; d[1] = (uint16_t)(lo >> 16); d[2] = (uint16_t)hi; d[3] = (uint16_t)(hi >> 16); }
        }
    }
    if (a.xq_out == nullptr && a.xh_out == nullptr) return;
    // as q80_block_store: scale from the block's largest magnitude, codes by its reciprocal
    float amax = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
#pragma unroll
    for (int w = 1; w < 8; w <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, w));
    const float d = amax / 127.0f, id = d != 0.0f ? 1.0f / d : 0.0f, df = __half2float(__float2half_rn(d));
    const int q[4] = {__float2int_rn(y.x * id), __float2int_rn(y.y * id), __float2int_rn(y.z * id), __float2int_rn(y.w * id)};
    const int kt = col >> 7, kb = (col >> 5) & 3, j = (col & 31) >> 2;
    if (a.xq_out != nullptr) {
        int sum = q[0] + q[1] + q[2] + q[3];
#pragma unroll
        for (int w = 1; w < 8; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (live) {
            uint8_t* row = a.xq_out + ((size_t)kt * a.out_mcap + m) * XQ_ROW_BYTES;
            *reinterpret_cast<uint32_t*>(row + kb * 32 + j * 4) = (uint32_t)(q[0] & 0xff) | ((uint32_t)(q[1] & 0xff) << 8) | ((uint32_t)(q[2] & 0xff) << 16) | ((uint32_t)(q[3] & 0xff) << 24);
            if (j == 0) {
                reinterpret_cast<float*>(row + 128)[kb] = df;
                reinterpret_cast<int*>(row + 144)[kb] = 8 * sum;
            }
        }
    }
    if (a.xh_out != nullptr && live) {
        const float dfh = fminf(df, 515.0f);
        const __half2 u = __floats2half2_rn((float)q[0] * dfh, (float)q[2] * dfh), v = __floats2half2_rn((float)q[1] * dfh, (float)q[3] * dfh);      // (K order of xh_slot)
        uint8_t* at = a.xh_out + ((size_t)kt * (a.out_mcap >> 3) + (m >> 3)) * XH_ROWGROUP_BYTES + (size_t)(kb * 4 + (j & 3)) * 128 + (m & 7) * 16 + (j >> 2) * 8;
        *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
    }
}

// ------------------------------------------------------------------------------------------------
// Decode rows: both products on mma.sync m16n8k32 with int8 operands: keys and values go in as they lie in the cache, nothing is widened, and sums are exact
// 32-bit integers.  What is f32 is taken as digits of base 256 in rows of the MMA's A operand:
//   a query   n = rint(q 8355000 / max|q|), three signed digits of a head in rows g, g + 8, g + 4 (24 bits of the head's largest value)
//   a weight  n = rint(p s_v 2^(22 - e)), three unsigned digits; e: exponent of the largest p s_v that the row has met (held like a softmax maximum: what
//             was summed is rescaled when it moves), s_v the value's scale.  So each weight is off by 2^-23 of the largest one at most, as a f32 sum is
// Four heads fill the 16 rows; more heads of a key/value head go to CTAs of their own, which find its pages in L2 (eight in two tiles of one CTA, 255 registers: one
// row of 30000 tokens 22.4 us for 19.7, 6 rows of 3000 13.9 for 12.6, 40 rows 53 for 47, with heads of 64 31 for 34).
//
// A warp takes a page (32 tokens) at a time through a private ring of cp.async stages, 16-byte pieces XOR-swizzled by the token so that both ldmatrix
// forms are free of conflicts: no barrier between warps until the final merge.
//
// What bounds it: the cache's bytes for long contexts, a chain of latencies for short ones.  32 rows of 1500 to 3000 tokens (8 kv heads of 128, 152 MB) 29.6
// us, 5.1 TB/s (the same loads without the arithmetic 27.3); one row of 100003 tokens 38.5 us, 5.5 TB/s; one of 192 tokens 4.5 us.  A page takes a warp 1240 clk from end to end (260 of them its 32 MMAs,
// 190 the special-function unit's 24 conversions and exponentials) and an SM with three CTAs 110.  Integer sums that stay in the accumulators from page to page take
// 3 % off that and put it back on in the end, where they are converted.  One CTA of eight warps per SM that walks an equal stretch of all
// rows' pages evens out the SMs' loads (256 CTAs on 148 SMs: 1.5 to 1), but every change of row empties its pipeline: 45 us.
// ------------------------------------------------------------------------------------------------
#define KA_WARPS 4
#define KA_MIN_SPLIT_PAGES 24        // contexts up to 768 tokens: no split
#define KA_MOST_CTAS 8               // of a cluster that shares a prompt tile's pages
#define KA_COUNTER_BYTES 65536       // completion counters at scratch offset 0 (dl_attention_scratch_bytes)

DL_DEVINL void ka_cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
DL_DEVINL void ka_ldm(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
// two 16 x 16 byte matrices, transposed: lane l gets rows 4 (l % 4) .. + 3 of columns l / 4 and l / 4 + 8 of the first, then of the second
DL_DEVINL void ka_ldm_bytes(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
DL_DEVINL void ka_mma_first(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
DL_DEVINL void ka_mma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};" : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DL_DEVINL void ka_mma_u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
DL_DEVINL void ka_mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};" : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DL_DEVINL float ka_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
DL_DEVINL float ka_max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// shift of a token's 16-byte pieces: tokens 2 j + {0, 1, 8, 9, 16, 17, 24, 25} (a column of scores for each lane) and {0 .. 3, 8 .. 11} + 4 i (a phase of the
// byte-wise ldmatrix) come to lie in eight different columns of 16 bytes (heads of 32: in four)
template <int HS> DL_DEVINL int ka_swizzle(int t) {
    const int f = (t & 1) | (((t >> 3) & 1) << 1) | ((((t >> 4) ^ (t >> 1)) & 1) << 2);
    return HS == 128 ? f : HS == 64 ? f >> 1 : f >> 2;
}

// a page of one key/value head into a stage: codes of the keys, of the values (swizzled), scales of both
template <int HS> struct KaStage {
    static constexpr int CODES = KV8_PAGE * HS, BYTES = 2 * CODES + 2 * KV8_PAGE * 4;
};
template <int HS> DL_DEVINL void ka_load(const DlKv8Cache& c, size_t line, uint32_t dst, int lane) {
    constexpr int CH = HS / 16, CODES = KaStage<HS>::CODES;
    const int8_t* ks = c.k + line * HS + lane * 16;
    const int8_t* vs = c.v + line * HS + lane * 16;
#pragma unroll
    for (int j = 0; j < CH; j++) {
        const int idx = j * 32 + lane, t = idx / CH, p = idx % CH;
        const uint32_t d = dst + t * HS + ((p ^ ka_swizzle<HS>(t)) << 4);
        ka_cp16(d, ks + j * 512);
        ka_cp16(d + CODES, vs + j * 512);
    }
    if (lane < 16) ka_cp16(dst + 2 * CODES + lane * 16, (lane < 8 ? c.k_scale : c.v_scale) + line + (lane & 7) * 4);
}
// the lane's share of a query: dimensions 16 k + 4 (lane % 4) .. + 3
template <int HS> DL_DEVINL void ka_query(const float* q, bool vec, float (&x)[HS / 16][4]) {
#pragma unroll
    for (int k = 0; k < HS / 16; k++) {
        if (vec) {
            const float4 v = *reinterpret_cast<const float4*>(q + k * 16);
            x[k][0] = v.x; x[k][1] = v.y; x[k][2] = v.z; x[k][3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[k][e] = q[k * 16 + e];
        }
    }
}
// ... as signed digits in the A fragments: THREE in rows g, g + 8 (lower) and g + 4 (the upper lanes' g), or two in rows g, g + 8.  Returns what an integer sum is
// multiplied with, log2(e) / sqrt(HS) in it: sums are c[g] 256 + c[g + 8], of the upper lanes 2^-16 of that
template <int HS, bool THREE> DL_DEVINL float ka_digits(const float (&x)[HS / 16][4], bool live, bool lower, uint32_t (&qf)[HS / 32][4]) {
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < HS / 16; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // (queries below 2^-100: their scores are zeros)
    const bool finite = top < 0x7f800000u, zero = !finite || __uint_as_float(top) < KV8_TINY || !live;
    constexpr float MOST = THREE ? 8355000.f : 32600.f;
    const float up = zero ? 0.f : MOST / __uint_as_float(top);
#pragma unroll
    for (int k = 0; k < HS / 16; k++) {
        uint32_t n[4];
#pragma unroll
        for (int e = 0; e < 4; e++) n[e] = (uint32_t)(zero ? 0 : __float2int_rn(x[k][e] * up));
        // signed digits: bytes of n + 0x80...80, each less 0x80
#pragma unroll
        for (int e = 0; e < 4; e++) n[e] = THREE ? (n[e] + 0x808080u) ^ 0x808080u : (n[e] + 0x8080u) ^ 0x8080u;
        const uint32_t sel = !THREE ? 0x4051u : lower ? 0x5162u : 0x5140u;
        const uint32_t u = __byte_perm(n[0], n[1], sel), v = __byte_perm(n[2], n[3], sel);
        qf[k / 2][(k & 1) * 2] = __byte_perm(u, v, 0x5410);
        qf[k / 2][(k & 1) * 2 + 1] = !THREE || lower ? __byte_perm(u, v, 0x7632) : 0u;
    }
    if (!finite && live) return __uint_as_float(0x7fffffffu);
    return zero ? 0.f : __uint_as_float(top) / MOST * (rsqrtf((float)HS) * 1.44269504088896341f) * (!THREE ? 1.f : lower ? 256.f : 1.f / 256.f);
}
// integer scores of a page.  Column n of score tile j is token 8 (n / 2) + 2 j + n % 2, so that a lane has the eight tokens 8 (lane % 4) .. + 7
template <int HS, int MT> DL_DEVINL void ka_scores(uint32_t kb, int lane, const uint32_t (&qf)[MT][HS / 32][4], int (&c)[MT][4][4]) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const int t = (((lane & 7) >> 1) << 3) + ((lane >> 4) << 1) + (lane & 1) + j * 2, piece = (lane >> 3) & 1;
        const uint32_t base = kb + t * HS, sw = ka_swizzle<HS>(t);
#pragma unroll
        for (int k = 0; k < HS / 32; k++) {
            uint32_t b[4];
            ka_ldm(b, base + (((2 * k + piece) ^ sw) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if (k == 0) {
                    ka_mma_first(c[mt][j], qf[mt][k], b[0], b[1]);
                    ka_mma_first(c[mt][j + 1], qf[mt][k], b[2], b[3]);
                } else {
                    ka_mma(c[mt][j], qf[mt][k], b[0], b[1]);
                    ka_mma(c[mt][j + 1], qf[mt][k], b[2], b[3]);
                }
            }
        }
    }
}
// the lane's row of the values' ldmatrix: k index 4 a + i of a product is token 8 a + i, k index 16 + 4 a + i token 8 a + 4 + i
DL_DEVINL int ka_value_row(int lane) { return (((lane & 15) >> 2) << 3) + (lane & 3) + ((lane >> 4) << 2); }
// scales of the lane's eight tokens
DL_DEVINL void ka_scales(const float* at, float (&s)[8]) {
    const float4 x = *reinterpret_cast<const float4*>(at), y = *reinterpret_cast<const float4*>(at + 4);
    s[0] = x.x; s[1] = x.y; s[2] = x.z; s[3] = x.w; s[4] = y.x; s[5] = y.y; s[6] = y.z; s[7] = y.w;
}
// The warps' sums in shared memory, rows 8 floats apart beyond their length: the eight rows that a warp's lanes store at once lie in different banks
template <int HS> struct KaSums { static constexpr int LD = HS + 8; };

struct Kv8Work {               // what the launch adds to the arguments of decode rows
    int n_splits, groups;      // shares of a row at most; CTAs that share a key/value head's query heads
    int shares;                // shares of rows beyond the first that the launch has room for
    float part;                // 1 / shares
    int least;                 // pages of a share at least
    unsigned* counters;        // [M][kv heads * groups]
    float* part_o;             // [M][heads][n_splits][HS]
    float* part_ml;            // [M][heads][n_splits][2]
};

// Rows share the launch's CTAs by their lengths: of all pages a share has P = pages / wk.shares, at least wk.least, and a row as many shares as it has P, whole ones,
// one at least.  So one user deep in a document beside others is not one CTA's per head (us with shares by the number of rows / so: 8 rows of 32 heads, one of 30000
// tokens, the others of 300: 29 / 15, 32 such rows 119 / 38), and rows of like lengths get about what they would get by their number (2 rows of 3000 8.5 / 9.4, 6 9.9 / 10.7,
// 12 12.9 / 13.2, 20 of 4000 28.2 / 27.3, 32 of 3000 29.9 / 29.2, 64 of 1500 33.3 / 33.3).
DL_DEVINL int ka_pages(const Kv8AttArgs& a, int m) {           // < 0: not this launch's row
    if (m >= a.rows.M || (a.row_skip != nullptr && a.row_skip[m] != 0)) return -1;
    const int t = kv8_tokens(a.rows, a.rows.pos[m], a.rows.slot[m]);
    return t > 0 ? (t - 1) / KV8_PAGE + 1 : 0;
}
// 1 / P, from all rows' pages
DL_DEVINL float ka_part(const Kv8Work& wk, unsigned total) { return __fdividef(1.f, fmaxf((float)wk.least, (float)total * wk.part)); }
// pages of all rows behind the first 32 that come to a lane
DL_DEVINL unsigned ka_rest(const Kv8AttArgs& a, int lane) {
    unsigned ours = 0;
#pragma unroll 4
    for (int base = 32; base < a.rows.M; base += 32) ours += max(ka_pages(a, base + lane), 0);
    return ours;
}
// whole parts, of eight pages begun ones (one less is below the quotient, so those beyond the rows' first are wk.shares at most, even if it is off a little: every
// warp finds the same numbers)
DL_DEVINL int ka_shares(const Kv8Work& wk, int pages, float part) {
    return pages <= KA_MIN_SPLIT_PAGES ? 1 : min(max((int)fmaf((float)pages, part, part == 0.125f ? 0.95f : 0.05f), 1), wk.n_splits);
}
// Of number idx among the shares that are not their row's first, in 32 rows whose shares the lanes have: row * 4096 + share * 64 + shares - 1, or -1 and idx less theirs
DL_DEVINL int ka_find(int n, int lane, int& idx) {
    int upto = n - 1;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
        const int ahead = __shfl_up_sync(0xffffffffu, upto, w);
        if (lane >= w) upto += ahead;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, upto > idx);
    const int l = hit != 0 ? __ffs(hit) - 1 : 31, found = l * 4096 + (idx - (upto - n + 1) + 1) * 64 + n - 1;
    idx -= __shfl_sync(0xffffffffu, upto, 31);
    return hit != 0 ? __shfl_sync(0xffffffffu, found, l) : -1;
}
// ... in more than 32 rows.  (Not inlined: what a launch of few rows does not run it does not fetch)
__device__ __noinline__ int ka_find_in_many(const Kv8AttArgs& a, const Kv8Work& wk, int idx, float part, int lane) {
    for (int base = 0; base < a.rows.M; base += 32) {
        const int found = ka_find(ka_shares(wk, ka_pages(a, base + lane), part), lane, idx);
        if (found >= 0) return base * 4096 + found;
    }
    return -1;
}

// grid (kv heads * groups, M + wk.shares): the rows' first shares, then the others
template <int HS, int ST>
__global__ void __launch_bounds__(KA_WARPS * 32) kv8_attention_kernel(const __grid_constant__ Kv8AttArgs a, const __grid_constant__ Kv8Work wk) {
    constexpr int CH = HS / 16, KS = HS / 32, NT = HS / 8, STAGE = KaStage<HS>::BYTES, CODES = KaStage<HS>::CODES;
    constexpr int SR = 4;                                                  // heads of the CTA
    constexpr int TOP = 22;                                                // a weight's integer is at most 2^(TOP + 1)
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, qd = lane & 3;
    const int kvh = blockIdx.x / wk.groups;
    const int G = a.heads / a.c.n_kv_heads, per = (G + wk.groups - 1) / wk.groups, h_lo = (blockIdx.x % wk.groups) * per, n_live = min(per, G - h_lo);
    const bool lower = g < 4;
    pdl_launch_dependents();
    pdl_wait();
    const int further = (int)blockIdx.y - a.rows.M;            // < 0: a row's first share
    const bool many = a.rows.M > 32, one = a.rows.M == 1;      // (one row: its number of shares hangs on nothing else; 0.7 us less than by the others' way)
    int m0 = further < 0 ? blockIdx.y : 0, sp = one ? blockIdx.y : 0, n_eff = 1;
    int mine = 0;                                              // pages of row `lane`, and of all rows that come to the lane
    unsigned ours = 0;
    auto all_rows = [&] {
        mine = ka_pages(a, lane);
        ours = max(mine, 0);
        if (many) ours += ka_rest(a, lane);
    };
    const bool at_once = wk.least == 8;                        // most rows will have several shares: asked for with this CTA's own position
    if (wk.n_splits > 1 && !one && (at_once || further >= 0)) all_rows();
    const int my_head = g & 3;
    float x[2 * KS][4];
    auto ask = [&] { ka_query<HS>(a.q + (size_t)m0 * a.ldq + (kvh * G + h_lo + (my_head < n_live ? my_head : 0)) * HS + qd * 4, ((uintptr_t)a.q & 15) == 0 && (a.ldq & 3) == 0, x); };
    if (further < 0 || one) {
        ask();                                                 // (ahead of what hangs on positions)
        if (a.row_skip != nullptr && a.row_skip[m0] != 0) return;
    } else {
        int idx = further;
        const float part = ka_part(wk, __reduce_add_sync(0xffffffffu, ours));
        const int found = many ? ka_find_in_many(a, wk, idx, part, lane) : ka_find(ka_shares(wk, mine, part), lane, idx);
        if (found < 0) return;
        m0 = found >> 12;
        sp = (found >> 6) & 63;
        n_eff = (found & 63) + 1;
        ask();
    }
    const int pos = a.rows.pos[m0], slot = a.rows.slot[m0];
    const int T0 = kv8_tokens(a.rows, pos, slot), T = max(T0, 0);
    bool bad = T0 < 0;
    const int n_pages = (T + KV8_PAGE - 1) / KV8_PAGE;
    if (one) {
        if (n_pages > KA_MIN_SPLIT_PAGES) n_eff = min(wk.n_splits, (n_pages + 7) / 8);
        if (sp >= n_eff) return;
    }
    const int pg0 = sp == 0 ? 0 : sp * ((n_pages + n_eff - 1) / n_eff);
    const int* bt = a.rows.block_table + (size_t)(bad ? 0 : slot) * a.rows.max_pages;
    auto page_at = [&](int i) {                                // page i of this warp: pg0 + warp + 4 i
        int p = pg0 + warp + KA_WARPS * i < n_pages ? bt[pg0 + warp + KA_WARPS * i] : 0;
        if ((unsigned)p >= (unsigned)a.rows.n_pages) { bad = true; p = 0; }
        return p;
    };
    int my_page = page_at(lane);                               // the lanes hold the next 32 page numbers
    const uint32_t ring = smem_u32(smem) + warp * (ST * STAGE);
    auto load = [&](int st, int page) { ka_load<HS>(a.c, ((size_t)page * a.c.n_kv_heads + kvh) * KV8_PAGE, ring + st * STAGE, lane); };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) {
        const int page = __shfl_sync(0xffffffffu, my_page, i);
        if (pg0 + warp + KA_WARPS * i < n_pages) load(i, page);            // (those of another share, where this one ends ahead of them, are not looked at)
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (further < 0 && !one && wk.n_splits > 1 && n_pages > max(KA_MIN_SPLIT_PAGES, wk.least)) {
        if (!at_once) all_rows();
        n_eff = ka_shares(wk, n_pages, ka_part(wk, __reduce_add_sync(0xffffffffu, ours)));
    }
    const int pps = n_eff == 1 ? n_pages : (n_pages + n_eff - 1) / n_eff, pg1 = min(n_pages, pg0 + pps), n_my = max(0, (pg1 - pg0 - warp + KA_WARPS - 1) / KA_WARPS);

    uint32_t qf[1][KS][4];
    const float fl = ka_digits<HS, true>(x, my_head < n_live, lower, qf[0]);
    float o[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) o[n][0] = o[n][1] = 0.f;
    float run_m = -INFINITY, run_l = 0.f, run_w = 0.f;         // maximum of scores, sum of weights (this lane's tokens), largest weight * scale
    int ex = 24;                                               // exponent field of run_w: the unit of o
    const uint32_t v_at = ka_value_row(lane) * HS, v_sw = ka_swizzle<HS>(ka_value_row(lane));

    int st = 0;
    for (int i = 0; i < n_my; i++) {
        {
            const int nx = i + ST - 1;
            if ((nx & 31) == 0) my_page = page_at(nx + lane);
            const int page = __shfl_sync(0xffffffffu, my_page, nx & 31);
            if (nx < n_my) load(st == 0 ? ST - 1 : st - 1, page);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        __syncwarp();
        const uint32_t kb = ring + st * STAGE, vb = kb + CODES;
        const float* scales = reinterpret_cast<const float*>(smem + (size_t)(warp * ST + st) * STAGE + 2 * CODES) + qd * 8;
        const int left = T - (pg0 + warp + KA_WARPS * i) * KV8_PAGE;
        float sk[8], sv[8];
        ka_scales(scales, sk);
        ka_scales(scales + KV8_PAGE, sv);
        int c[1][4][4];
        ka_scores<HS, 1>(kb, lane, qf, c);
        uint32_t vf[CH][4];                                    // (asked for ahead of the weights)
#pragma unroll
        for (int ch = 0; ch < CH; ch++) ka_ldm_bytes(vf[ch], vb + v_at + ((ch ^ v_sw) << 4));
        uint32_t pa[4];
        float s[8], w[8], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            s[e] = (float)(c[0][e >> 1][e & 1] * 256 + c[0][e >> 1][(e & 1) + 2]) * fl;
            s[e] += __shfl_xor_sync(0xffffffffu, s[e], 16);
            s[e] *= sk[e];
            w[e] = sv[e];
        }
        if (left < KV8_PAGE) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (qd * 8 + e >= left) { s[e] = -INFINITY; w[e] = 0.f; }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(run_m, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float corr = ka_exp2(run_m - m_use);
        run_m = m_new;
        float sum = 0.f, big = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = ka_exp2(s[e] - m_use);
            sum += p;
            w[e] *= p;
            big = ka_max_nan(big, w[e]);
        }
        run_l = fmaf(run_l, corr, sum);
        big = ka_max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = ka_max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
        big = ka_max_nan(big, run_w * corr);
        run_w = big;
        const int e_new = min(max((int)(__float_as_uint(big) >> 23), 24), 254);
        const float up = __uint_as_float((uint32_t)(TOP + 254 - e_new) << 23);
        float f = corr * __uint_as_float((uint32_t)(ex - TOP) << 23) * up;
        if (big != big) f = big;
        ex = e_new;
        uint32_t n[8];
#pragma unroll
        for (int e = 0; e < 8; e++) n[e] = __float_as_uint(fmaf(w[e], up, 8388608.f));     // the integer in the low 23 bits (and 2^23 itself as its top byte)
        const uint32_t sel = lower ? 0x5162u : 0x5140u;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t y = __byte_perm(n[4 * u], n[4 * u + 1], sel), z = __byte_perm(n[4 * u + 2], n[4 * u + 3], sel);
            pa[2 * u] = __byte_perm(y, z, 0x5410);
            pa[2 * u + 1] = lower ? __byte_perm(y, z, 0x7632) : 0u;
        }
#pragma unroll
        for (int ch = 0; ch < CH; ch++) {
            int y[4], z[4];
            ka_mma_u8(y, pa, vf[ch][0], vf[ch][2]);
            ka_mma_u8(z, pa, vf[ch][1], vf[ch][3]);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                o[2 * ch][e] = fmaf(o[2 * ch][e], f, (float)(y[e] * 256 + y[e + 2]));
                o[2 * ch + 1][e] = fmaf(o[2 * ch + 1][e], f, (float)(z[e] * 256 + z[e + 2]));
            }
        }
        __syncwarp();
        st = st == ST - 1 ? 0 : st + 1;
    }
    bad = __any_sync(0xffffffffu, bad);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                           // the ring is done with
    constexpr int LD = KaSums<HS>::LD, LPH = HS / 4, ZP = 32 / LPH;        // LPH lanes take a head
    float* w_acc = reinterpret_cast<float*>(smem);             // [WARPS][SR][LD]
    float* w_ml = w_acc + KA_WARPS * SR * LD;                  // [WARPS][SR][2]
    int* s_last = reinterpret_cast<int*>(w_ml + KA_WARPS * SR * 2);
    run_l += __shfl_xor_sync(0xffffffffu, run_l, 1);
    run_l += __shfl_xor_sync(0xffffffffu, run_l, 2);
    if (bad) run_l = __uint_as_float(0x7fffffffu);
    const float unit = __uint_as_float((uint32_t)(ex - TOP) << 23) * (lower ? 256.f : 1.f / 256.f);
    const int s = warp * SR + my_head;
    // the upper lanes' digits go to the lower ones, which take the even n-tiles; and the other way round
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float x0 = o[n][e] * unit, x1 = o[n + 1][e] * unit;
            v[e] = (lower ? x0 : x1) + __shfl_xor_sync(0xffffffffu, lower ? x1 : x0, 16);
        }
        *reinterpret_cast<float2*>(w_acc + s * LD + qd * 2 + (lower ? n : n + 1) * 8) = make_float2(v[0], v[1]);
    }
    if (lower && qd == 0) { w_ml[s * 2] = run_m; w_ml[s * 2 + 1] = run_l; }
    __syncthreads();
    const bool single = n_eff == 1;
    for (int base = warp * 32; base < n_live * LPH; base += KA_WARPS * 32) {       // a lane takes four dimensions of a head
        const int s = min((base + lane) / LPH, n_live - 1), d = lane % LPH * 4, hd = kvh * G + h_lo + s;
        const bool live = base + lane < n_live * LPH;
        float mw[KA_WARPS], Mx = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) { mw[w] = w_ml[(w * SR + s) * 2]; Mx = fmaxf(Mx, mw[w]); }
        const float Mu = Mx == -INFINITY ? 0.f : Mx;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) {
            const float e = ka_exp2(mw[w] - Mu);
            const float4 x = *reinterpret_cast<const float4*>(w_acc + (w * SR + s) * LD + d);
            L = fmaf(w_ml[(w * SR + s) * 2 + 1], e, L);
            O.x = fmaf(x.x, e, O.x); O.y = fmaf(x.y, e, O.y); O.z = fmaf(x.z, e, O.z); O.w = fmaf(x.w, e, O.w);
        }
        if (single) {
            const float inv = L == 0.f && T == 0 ? 0.f : 1.f / L;
            kv8_store4(a, m0, hd * HS + d, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv), live, lane);
        } else if (live) {
            const size_t pidx = ((size_t)m0 * a.heads + hd) * wk.n_splits + sp;
            *reinterpret_cast<float4*>(wk.part_o + pidx * HS + d) = O;
            if (d == 0) { wk.part_ml[pidx * 2] = Mx; wk.part_ml[pidx * 2 + 1] = L; }
        }
    }
    if (single) return;
    __syncthreads();
    if (tid == 0) {                                            // the CTA's sums, ahead of the barrier, are released with its count
        unsigned* counter = &wk.counters[m0 * gridDim.x + blockIdx.x];
        unsigned prev;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(prev) : "l"(counter) : "memory");
        *s_last = prev == (unsigned)n_eff - 1u ? 1 : 0;
        if (*s_last) *counter = 0u;
    }
    __syncthreads();
    if (!*s_last) return;
    // a warp merges a head: the lanes hold the splits' (max, sum); then HS / 4 lanes take a split's sums, 32 / (HS / 4) splits side by side, eight of each in flight
    for (int s = warp; s < n_live; s += KA_WARPS) {
        const int hd = kvh * G + h_lo + s;
        const size_t base = ((size_t)m0 * a.heads + hd) * wk.n_splits;
        float mz[2], lz[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int z = u * 32 + lane;
            mz[u] = z < n_eff ? __ldcg(&wk.part_ml[(base + z) * 2]) : -INFINITY;
            lz[u] = z < n_eff ? __ldcg(&wk.part_ml[(base + z) * 2 + 1]) : 0.f;
        }
        const float Mx = warp_max(fmaxf(mz[0], mz[1])), Mu = Mx == -INFINITY ? 0.f : Mx;
#pragma unroll
        for (int u = 0; u < 2; u++) mz[u] = ka_exp2(mz[u] - Mu);
        const float L = warp_sum(fmaf(lz[0], mz[0], lz[1] * mz[1]));
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* src = wk.part_o + base * HS + lane % LPH * 4;
        for (int z0 = 0; z0 < n_eff; z0 += 8 * ZP) {
            float4 x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int z = z0 + u * ZP + lane / LPH;
                x[u] = z < n_eff ? __ldcg(reinterpret_cast<const float4*>(src + (size_t)z * HS)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int z = z0 + u * ZP + lane / LPH;
                const float e0 = __shfl_sync(0xffffffffu, mz[0], z & 31), e1 = __shfl_sync(0xffffffffu, mz[1], z & 31), e = z < 32 ? e0 : e1;
                O.x = fmaf(x[u].x, e, O.x); O.y = fmaf(x[u].y, e, O.y); O.z = fmaf(x[u].z, e, O.z); O.w = fmaf(x[u].w, e, O.w);
            }
        }
#pragma unroll
        for (int w = LPH; w < 32; w <<= 1) {
            O.x += __shfl_xor_sync(0xffffffffu, O.x, w); O.y += __shfl_xor_sync(0xffffffffu, O.y, w);
            O.z += __shfl_xor_sync(0xffffffffu, O.z, w); O.w += __shfl_xor_sync(0xffffffffu, O.w, w);
        }
        const float inv = 1.f / L;
        kv8_store4(a, m0, hd * HS + lane % LPH * 4, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv), lane < LPH, lane);
    }
}

// ------------------------------------------------------------------------------------------------
// Prompt chunks: eight (row, head) pairs of one key/value head, of two digits a query (16 bits), fill an int8 MMA, two of them make the 16 rows of a tile, whose
// pages four warps share.  Two digits of a weight would not do: what is below 2^-16 of the largest weight is lost, however many tokens there are.  So
// weights p s_v are fp16 here, in a unit by the row's largest one that still counts (2^-11 of themselves, below 2^-20 of the largest 2^-31 of that), values are widened
// in registers -- codes are exact in fp16 -- and sums are the f32 accumulators of m16n8k16.
// p = 2^(s - ref) goes by a reference that moves only when a score is more than 2^8 above it, the unit only then or when a weight outgrows fp16: a vote of the warp, so
// that a page in the steady state takes no exchange for a running maximum and no rescaling.
//
// What bounds it: a warp's chain of latencies through a page, with two warps of 221 registers on each scheduler (64 MMAs a page, the tensor pipe is active 21 % of
// the SMs' time, a third of the clocks issue).  100 rows of 32 heads on 8 of 128 behind 1000 tokens 18.3 to 19.3 us, 200 of 64 behind 1000 21, 500 of 32 behind 500 24.6.
// Against 64 bits 2.1e-4 of a row's size (f32 rows, 130 behind 1000).  32 stacked rows a CTA, which halves the
// widening, takes 34 % more for 30 rows of heads of 64 behind 1000 tokens (there are half the CTAs) and as much for 200; the next page's scores ahead of this one's
// products spill.
// ------------------------------------------------------------------------------------------------
template <int HS, int ST>
__global__ void __launch_bounds__(KA_WARPS * 32, HS == 128 ? 2 : 4) kv8_prompt_kernel(const __grid_constant__ Kv8AttArgs a) {
    constexpr int CH = HS / 16, KS = HS / 32, NT = HS / 8, STAGE = KaStage<HS>::BYTES, CODES = KaStage<HS>::CODES;
    constexpr int SR = 16;                                                 // stacked rows of the CTA
    constexpr int TOP = 6;                                                 // the largest weight is below 2^(TOP + 1) units when the unit is chosen,
    constexpr float MOST_W = 0x1p15f, AHEAD = 8.f;                         // and below this always; scores may pass the reference by so much (log2)
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, qd = lane & 3;
    const int kvh = blockIdx.y, G = a.heads / a.c.n_kv_heads;
    uint32_t n_cta, rank;                                      // CTAs of the cluster: they share the tile's pages
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n_cta));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    pdl_launch_dependents();
    pdl_wait();
    // stacked row s of the tile is pair s_lo + s = row * G + head of the group, row 0 (batch row m0) at position p0
    int tile = (gridDim.x - 1 - blockIdx.x) / n_cta, m0 = 0, end = 0;      // late tiles (long histories) first
    {
        const int mine = lane < 17 ? a.meta[min(lane, 2 * min(max(a.meta[0], 0), a.n_seg))] : 0;      // (what lies behind the last segment is not read)
        const int n_seg = min(__shfl_sync(0xffffffffu, mine, 0), a.n_seg);
        int i = 0;
        for (; i < n_seg; i++) {
            m0 = __shfl_sync(0xffffffffu, mine, 1 + 2 * i);
            end = __shfl_sync(0xffffffffu, mine, 2 + 2 * i);
            if (m0 < 0 || end > a.rows.M || end <= m0) continue;
            const int nt = ((end - m0) * G + SR - 1) / SR;
            if (tile < nt) break;
            tile -= nt;
        }
        if (i >= n_seg) return;
    }
    const int s_lo = tile * SR, n_live = min(SR, (end - m0) * G - s_lo), p0 = a.rows.pos[m0], slot = a.rows.slot[m0];
    auto row_of = [&](int s) { return m0 + (s_lo + s) / G; };
    auto head_of = [&](int s) { return kvh * G + (s_lo + s) % G; };
    float x[2][2 * KS][4];
#pragma unroll
    for (int mt = 0; mt < 2; mt++) {
        const int s = mt * 8 + g < n_live ? mt * 8 + g : 0;
        ka_query<HS>(a.q + (size_t)row_of(s) * a.ldq + head_of(s) * HS + qd * 4, ((uintptr_t)a.q & 15) == 0 && (a.ldq & 3) == 0, x[mt]);
    }
    bool bad = p0 >= 0 && (p0 > 0x7fffffff - (end - m0) || kv8_tokens(a.rows, p0 + (end - m0) - 1, slot) < 0);
    const int T = bad || p0 < 0 ? 0 : p0 + (s_lo + n_live - 1) / G + 1, all = min(T, p0 + s_lo / G + 1);       // tokens that the last, that every row of the tile sees
    if ((T + KV8_PAGE - 1) / KV8_PAGE < 8 * (int)n_cta) {      // too few pages to share: the first CTA's
        if (rank > 0) return;
        n_cta = 1;
    }
    const int step = KA_WARPS * n_cta, w0 = rank * KA_WARPS + warp, n_pages = (T + KV8_PAGE - 1) / KV8_PAGE, n_my = max(0, (n_pages - w0 + step - 1) / step);      // this warp's pages: w0 + step i
    const int* bt = a.rows.block_table + (size_t)(bad ? 0 : slot) * a.rows.max_pages;

    const uint32_t ring = smem_u32(smem) + warp * (ST * STAGE);
    auto page_at = [&](int i) {
        int p = i < n_my ? bt[w0 + step * i] : 0;
        if ((unsigned)p >= (unsigned)a.rows.n_pages) { bad = true; p = 0; }
        return p;
    };
    int my_page = page_at(lane);                               // the lanes hold the next 32 page numbers
    auto load = [&](int st, int page) { ka_load<HS>(a.c, ((size_t)page * a.c.n_kv_heads + kvh) * KV8_PAGE, ring + st * STAGE, lane); };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) {
        const int page = __shfl_sync(0xffffffffu, my_page, i);
        if (i < n_my) load(i, page);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    uint32_t qf[2][KS][4];
    float fl[2], ref[2], run_l[2], run_w[2], up[2];            // reference of the weights, their sum and largest weight * scale (this lane's tokens), their unit's inverse
    int lim[2];                                                // tokens that the lane's rows see
#pragma unroll
    for (int mt = 0; mt < 2; mt++) {
        const int s = mt * 8 + g;
        fl[mt] = ka_digits<HS, false>(x[mt], s < n_live, true, qf[mt]);
        lim[mt] = s < n_live ? min(T, p0 + (s_lo + s) / G + 1) : 0;
        ref[mt] = -INFINITY;
        run_l[mt] = run_w[mt] = 0.f;
        up[mt] = 0x1p109f;
    }
    float o[NT][4];                                            // rows g (0, 1) and g + 8 (2, 3)
#pragma unroll
    for (int n = 0; n < NT; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    const auto rescale = [&](float c0, float c1) {
#pragma unroll
        for (int n = 0; n < NT; n++) { o[n][0] *= c0; o[n][1] *= c0; o[n][2] *= c1; o[n][3] *= c1; }
    };
    const uint32_t v_at = ka_value_row(lane) * HS, v_sw = ka_swizzle<HS>(ka_value_row(lane));

    int st = 0;
    for (int i = 0; i < n_my; i++) {
        {
            const int nx = i + ST - 1;
            if ((nx & 31) == 0) my_page = page_at(nx + lane);
            const int page = __shfl_sync(0xffffffffu, my_page, nx & 31);
            if (nx < n_my) load(st == 0 ? ST - 1 : st - 1, page);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        __syncwarp();
        const uint32_t kb = ring + st * STAGE, vb = kb + CODES;
        const float* scales = reinterpret_cast<const float*>(smem + (size_t)(warp * ST + st) * STAGE + 2 * CODES) + qd * 8;
        const int tok0 = (w0 + step * i) * KV8_PAGE;
        float sk[8], sv[8], s[2][8], w[2][8], top[2];
        ka_scales(scales, sk);
        ka_scales(scales + KV8_PAGE, sv);
        int c[2][4][4];
        ka_scores<HS, 2>(kb, lane, qf, c);
        bool move = false;
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                s[mt][e] = (float)(c[mt][e >> 1][e & 1] * 256 + c[mt][e >> 1][(e & 1) + 2]) * fl[mt] * sk[e];
                w[mt][e] = sv[e];
            }
            if (tok0 + KV8_PAGE > all) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (tok0 + qd * 8 + e >= lim[mt]) { s[mt][e] = -INFINITY; w[mt][e] = 0.f; }
            }
            top[mt] = s[mt][0];
#pragma unroll
            for (int e = 1; e < 8; e++) top[mt] = fmaxf(top[mt], s[mt][e]);
            move |= top[mt] > ref[mt] + AHEAD;
        }
        float corr[2] = {1.f, 1.f};
        bool unit = __any_sync(0xffffffffu, move);
        if (unit) {                                            // the references move to the maxima
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                top[mt] = fmaxf(top[mt], __shfl_xor_sync(0xffffffffu, top[mt], 1));
                top[mt] = fmaxf(top[mt], __shfl_xor_sync(0xffffffffu, top[mt], 2));
                top[mt] = fmaxf(top[mt], ref[mt]);
                corr[mt] = ref[mt] == -INFINITY ? 0.f : ka_exp2(ref[mt] - top[mt]);
                ref[mt] = top[mt];
                run_l[mt] *= corr[mt];
                run_w[mt] *= corr[mt];
            }
        }
        bool grow = false;
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            const float m = ref[mt] == -INFINITY ? 0.f : ref[mt];
            float sum = 0.f;
            top[mt] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = ka_exp2(s[mt][e] - m);
                sum += p;
                w[mt][e] *= p;
                top[mt] = ka_max_nan(top[mt], w[mt][e]);
            }
            run_l[mt] += sum;
            run_w[mt] = ka_max_nan(run_w[mt], top[mt]);
            grow |= !(top[mt] * up[mt] < MOST_W);
        }
        unit |= __any_sync(0xffffffffu, grow);
        if (unit) {                                            // another unit: weights have grown, or the largest ones count less beside the new maxima (or a NaN)
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                float big = ka_max_nan(run_w[mt], __shfl_xor_sync(0xffffffffu, run_w[mt], 1));
                big = ka_max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
                if (!(big < INFINITY)) run_l[mt] = __uint_as_float(0x7fffffffu);
                else {
                    const float now = __uint_as_float((uint32_t)(TOP + 254 - min(max((int)(__float_as_uint(big) >> 23), 24), 254)) << 23);
                    corr[mt] = corr[mt] * (1.f / up[mt]) * now;      // (2 at most, as what counted before counts in `big`)
                    up[mt] = now;
                }
            }
            rescale(corr[0], corr[1]);
        }
        // values of 8 tokens for each lane: k index 2 a, 2 a + 1, 8 + 2 a, 9 + 2 a of an MMA are tokens 8 a .. + 3, of the next one 8 a + 4 .. + 7
        uint32_t pa[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int u = 0; u < 4; u++) {                      // row g, row g + 8, then the same of the next two tokens
                const int e = h * 4 + (u >> 1) * 2;
                const __half2 y = __floats2half2_rn(w[u & 1][e] * up[u & 1], w[u & 1][e + 1] * up[u & 1]);
                pa[h][u] = *reinterpret_cast<const uint32_t*>(&y);
            }
#pragma unroll
        for (int ch = 0; ch < CH; ch++) {
            uint32_t b[4];
            ka_ldm_bytes(b, vb + v_at + ((ch ^ v_sw) << 4));
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int u = 0; u < 2; u++) {                  // 1024 + 128 + code as fp16, less 1152
                    const uint32_t y = b[h * 2 + u] ^ 0x80808080u;
                    uint32_t lo = __byte_perm(y, 0x64646464u, 0x4140), hi = __byte_perm(y, 0x64646464u, 0x4342);
                    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x64806480u));
                    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x64806480u));
                    ka_mma_f16(o[2 * ch + u], pa[h], lo, hi);
                }
        }
        __syncwarp();
        st = st == ST - 1 ? 0 : st + 1;
    }
    bad = __any_sync(0xffffffffu, bad);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                           // the ring is done with
    constexpr int LD = KaSums<HS>::LD, LPH = HS / 4;           // LPH lanes take a row
    float* w_acc = reinterpret_cast<float*>(smem);             // [WARPS][SR][LD]
    float* w_ml = w_acc + KA_WARPS * SR * LD;                  // [WARPS][SR][2]
    float* share = w_ml + KA_WARPS * SR * 2;                   // [SR][WARPS * CTAs]: what a row's sums count
    int* place = reinterpret_cast<int*>(share + SR * KA_WARPS * KA_MOST_CTAS);     // [SR][2]: batch row, first column
    rescale(1.f / up[0], 1.f / up[1]);
#pragma unroll
    for (int mt = 0; mt < 2; mt++) {
        run_l[mt] += __shfl_xor_sync(0xffffffffu, run_l[mt], 1);
        run_l[mt] += __shfl_xor_sync(0xffffffffu, run_l[mt], 2);
        if (bad) run_l[mt] = __uint_as_float(0x7fffffffu);
        const int s = warp * SR + mt * 8 + g;
#pragma unroll
        for (int n = 0; n < NT; n++) *reinterpret_cast<float2*>(w_acc + s * LD + qd * 2 + n * 8) = make_float2(o[n][2 * mt], o[n][2 * mt + 1]);
        if (qd == 0) { w_ml[s * 2] = ref[mt]; w_ml[s * 2 + 1] = run_l[mt]; }
    }
    // every CTA of the cluster sums its share of the tile's rows over all of them
    cg::cluster_group cluster = cg::this_cluster();
    if (n_cta > 1) cluster.sync();
    else __syncthreads();
    const int mine = n_live > (int)rank ? (n_live - 1 - (int)rank) / (int)n_cta + 1 : 0;       // rows rank, rank + n_cta, ...
    const int parts = KA_WARPS * n_cta;                        // (a power of two, 32 at most: a row's lanes lie in one warp)
    if (warp < 2) {
        const int j = tid / parts, z = tid % parts, s = rank + j * n_cta;
        float m = -INFINITY, l = 0.f;
        if (j < mine) {
            const float* ml = cluster.map_shared_rank(w_ml, z / KA_WARPS) + ((z % KA_WARPS) * SR + s) * 2;
            m = ml[0];
            l = ml[1];
        }
        float Mx = m;
        for (int w = 1; w < parts; w <<= 1) Mx = fmaxf(Mx, __shfl_xor_sync(0xffffffffu, Mx, w));
        const float e = ka_exp2(m - (Mx == -INFINITY ? 0.f : Mx));
        float L = l * e;
        for (int w = 1; w < parts; w <<= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
        if (j < mine) {
            share[tid] = L == 0.f && T == 0 ? 0.f : e / L;
            if (z == 0) { place[j * 2] = row_of(s); place[j * 2 + 1] = head_of(s) * HS; }
        }
    }
    __syncthreads();
    for (int base = warp * 32; base < mine * LPH; base += KA_WARPS * 32) {         // a lane takes four dimensions of a row
        const int j = min((base + lane) / LPH, mine - 1), s = rank + j * n_cta, d = lane % LPH * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t r = 0; r < n_cta; r++) {
            const float* from = cluster.map_shared_rank(w_acc, r) + s * LD + d;
            const float4 e4 = *reinterpret_cast<const float4*>(share + j * parts + r * KA_WARPS);
            const float e[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
            for (int w = 0; w < KA_WARPS; w++) {
                const float4 x = *reinterpret_cast<const float4*>(from + w * SR * LD);
                y.x = fmaf(x.x, e[w], y.x); y.y = fmaf(x.y, e[w], y.y); y.z = fmaf(x.z, e[w], y.z); y.w = fmaf(x.w, e[w], y.w);
            }
        }
        kv8_store4(a, place[j * 2], place[j * 2 + 1] + d, y, base + lane < mine * LPH, lane);
    }
    if (n_cta > 1) cluster.sync();                             // (no CTA leaves while its sums are read)
}

template <typename K, typename... A>
static int ka_launch(const char* who, K kernel, SmemLimit& given, dim3 grid, int cluster, int threads, int smem, int pdl, void* stream, const A&... args) {
    if (const int rc = smem > 0 ? dl_smem_limit(who, kernel, smem, given) : 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        cfg.numAttrs++;
    }
    if (pdl) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) { dl_set_error("%s launch: %s", who, cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

template <int HS>
static int ka_decode(const Kv8AttArgs& a, int n_splits, void* scratch, int pdl, void* stream) {
    constexpr int ST = 256 / HS, smem = KA_WARPS * ST * KaStage<HS>::BYTES;
    static_assert(KA_WARPS * 4 * (KaSums<HS>::LD + 2) * 4 + 4 <= smem, "the merge fits the ring");
    static SmemLimit given;
    const int kv = a.c.n_kv_heads, G = a.heads / kv, M = a.rows.M;
    Kv8Work wk = {n_splits, (G + 3) / 4, 0, 0.f, 8, nullptr, nullptr, nullptr};
    // CTAs: as many as the SMs hold with some to spare, more where those of one key/value head read the same pages.  8 kv heads of 128, rows of one length, us with
    // one share each / these / about twice as many: one row of 100003 tokens 528 / 38.5 / 54, 6 rows of 3000 20 / 10.1 / 13.3, 12 rows of 3000 19.7 / 15.8 / 20, 20 rows of
    // 4000 30.8 / 28.1 / 30.3, 32 rows of 3000 29.7 / 29.7 / 37; eight heads for each: one row of 30000 165 / 20 / 23.5, 7 of 5000 24 / 17.5 / 20, of heads of 64 18 /
    // 13.1 / 15.6
    // Where the rows alone take three quarters of them, 64 more, for rows that are much longer than the others, of 64 pages each or more: 128 cost 32 rows of 3000 that
    // have no use for them 0.4 us more, and summing up all rows' pages in every CTA 0.8 more
    const int unit = kv * wk.groups, ctas = wk.groups == 1 ? 320 : 400;
    const bool full = 4LL * M * unit >= 3 * ctas;
    wk.shares = max(1, (full ? 64 : ctas) / unit);
    if (full) wk.least = 64;
    wk.part = 1.f / wk.shares;
    if (n_splits > 1) {
        if ((long long)M * kv * wk.groups * 4 > KA_COUNTER_BYTES) { dl_set_error("dl_kv8_attention: M*n_kv_heads too large for splits"); return -1; }
        uint8_t* at = reinterpret_cast<uint8_t*>(scratch);
        wk.counters = reinterpret_cast<unsigned*>(at);
        wk.part_o = reinterpret_cast<float*>(at + KA_COUNTER_BYTES);
        wk.part_ml = reinterpret_cast<float*>(at + KA_COUNTER_BYTES + ((long long)M * a.heads * n_splits * HS * 4 + 255) / 256 * 256);
    }
    if (M == 1 && wk.n_splits > wk.shares) wk.n_splits = wk.shares;
    const unsigned rows = wk.n_splits == 1 ? M : min((long long)M + wk.shares, (long long)M * wk.n_splits);
    return ka_launch("dl_kv8_attention", kv8_attention_kernel<HS, ST>, given, dim3(kv * wk.groups, rows), 1, KA_WARPS * 32, smem, pdl, stream, a, wk);
}
template <int HS>
static int ka_prompt(const Kv8AttArgs& a, int pdl, void* stream) {
    constexpr int ST = HS == 32 ? 4 : 2, ring = KA_WARPS * ST * KaStage<HS>::BYTES, merge = 16 * (KA_WARPS * (KaSums<HS>::LD + 2 + KA_MOST_CTAS) + 2) * 4, smem = ring > merge ? ring : merge;
    const long long tiles = ((long long)a.rows.M * (a.heads / a.c.n_kv_heads) + 15) / 16 + 8;        // upper bound of the tiles of all segments
    static SmemLimit given;
    // CTAs of a tile where tiles leave SMs idle (us with one / two / four: 32 tiles behind 3000 tokens 31 / 25 / 23, behind none 8.1 / 8.6 / 9.2; 64 behind 1000 15.7 /
    // 14.7 / 15.6; 128 behind 2000 30.2 / 25.6 / 31.3, behind 500 14.4 / 14.9 / 24; 200 behind 1000 20.1 / 19.2 / 31, behind none 9.1 / 10.6 / 16)
    const long long ctas = (tiles - 8) * a.c.n_kv_heads;
    const int cluster = ctas <= 40 ? 4 : ctas <= 160 ? 2 : 1;
    return ka_launch("dl_kv8_attention_prefill", kv8_prompt_kernel<HS, ST>, given, dim3((unsigned)tiles * cluster, a.c.n_kv_heads), cluster, KA_WARPS * 32, smem, pdl, stream, a);
}

// ------------------------------------------------------------------------------------------------
// Long prompt chunks of heads of 64 and 128: the segments' pages widened once to fp16 (fp16(code * scale): 2^-11 of a value at most, the queries of that kernel are rounded alike),
// then the tcgen05 kernel of the fp16 cache on them, under the same page numbers.  Widening inside that kernel would be done again by every CTA that meets a page
// (rows / 128 * heads / 2 of them).  4001 rows behind 77 tokens: 8 MB in and 17 MB out, beside 136 GFLOP; both kernels 144 to 150 us, 910 to 945 TFLOP/s (172 with inputs in turn).
// Against 64 bits 5.4e-4 of a row's size (f32 rows, 130 behind 1000).
// Eight lanes list a segment each: one thread after the other, and every CTA for pages that are not there, took 0.8 us more.
//
// A line with a NaN (of the key or the value) becomes a key of NaN and a value of zeros: the rows that see it give NaN, and the weights of 0 that others
// have for it do not.  Values beyond fp16's range saturate.  What that kernel does not look at is looked at here: the segments that are in the tables are listed
// for it, rows of the others get NaN.
// ------------------------------------------------------------------------------------------------
struct Kv8ExpandArgs {
    Kv8AttArgs a;
    __half* k16;               // [pages][kv][32][HS]
    __half* v16;
    int* meta_out;             // [17]
};

template <int HS>
__global__ void __launch_bounds__(256) kv8_expand_kernel(const __grid_constant__ Kv8ExpandArgs x) {
    __shared__ int first[9], seg[8][3];                        // items ahead of a segment; begin, end, slot
    __shared__ int ok[8];
    const int tid = threadIdx.x, kv = x.a.c.n_kv_heads;
    pdl_launch_dependents();
    pdl_wait();
    if (tid < 8) {                                             // a lane for each segment
        const int n = max(0, min(x.a.meta[0], x.a.n_seg));
        const int b = tid < n ? x.a.meta[1 + 2 * tid] : 0, e = tid < n ? x.a.meta[2 + 2 * tid] : 0;
        const bool rows = b >= 0 && e <= x.a.rows.M && e > b;
        const int p = rows ? x.a.rows.pos[b] : 0, s = rows ? x.a.rows.slot[b] : 0;
        const bool there = rows && p >= 0 && p <= 0x7fffffff - (e - b) && kv8_tokens(x.a.rows, p + (e - b) - 1, s) > 0;
        int upto = there ? (p + (e - b) + KV8_PAGE - 1) / KV8_PAGE * kv : 0;
#pragma unroll
        for (int w = 1; w < 8; w <<= 1) {
            const int ahead = __shfl_up_sync(0xffu, upto, w);
            if (tid >= w) upto += ahead;
        }
        if (tid == 0) first[0] = 0;
        first[tid + 1] = upto;
        seg[tid][0] = b; seg[tid][1] = rows ? e : b; seg[tid][2] = s;
        ok[tid] = there;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        // pages that are not there: this CTA, which lists the segments, takes theirs as one that is not in the tables
        for (int i = 0; i < 8; i++) {
            if (first[i + 1] == first[i]) continue;
            const int* bt = x.a.rows.block_table + (size_t)seg[i][2] * x.a.rows.max_pages;
            const int pages = (first[i + 1] - first[i]) / kv;
            bool bad = false;
            for (int p = tid; p < pages; p += 256) bad |= (unsigned)bt[p] >= (unsigned)x.a.rows.n_pages;
            if (__syncthreads_or(bad) && tid == 0) ok[i] = 0;
        }
        __syncthreads();
    }
    if (blockIdx.x == 0) {
        if (tid == 0) {
            int n = 0;
            for (int i = 0; i < 8; i++)
                if (ok[i]) { x.meta_out[1 + 2 * n] = seg[i][0]; x.meta_out[2 + 2 * n] = seg[i][1]; n++; }
            x.meta_out[0] = n;
        }
        const int cols = x.a.heads * HS;
        for (int i = 0; i < 8; i++) {
            if (ok[i] || seg[i][1] <= seg[i][0]) continue;
            const float none = x.a.rows.pos[seg[i][0]] < 0 ? 0.f : __uint_as_float(0x7fffffffu);      // (rows without tokens)
            for (int m = seg[i][0] + (tid >> 5); m < seg[i][1]; m += 8)
                for (int c = tid & 31; c < cols; c += 32) {
                    kv8_store_y(x.a, m, c, none);
                    if (x.a.xq_out != nullptr || x.a.xh_out != nullptr) q80_block_store(none, tid & 31, m, c >> 5, x.a.out_mcap, x.a.xq_out, x.a.xh_out);
                }
        }
    }
    for (int item = blockIdx.x; item < first[8]; item += gridDim.x) {
        int i = 0;
        while (item >= first[i + 1]) i++;
        const int in = item - first[i], kvh = in % kv;
        const int page = x.a.rows.block_table[(size_t)seg[i][2] * x.a.rows.max_pages + in / kv];
        if ((unsigned)page >= (unsigned)x.a.rows.n_pages) continue;
        auto widen = [](uint4 c, float s, __half* dst) {
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float f[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    f[u] = (float)(int8_t)(w[e / 4] >> (8 * ((e + u) % 4))) * s;
                    f[u] = f[u] != f[u] ? f[u] : fminf(fmaxf(f[u], -65504.f), 65504.f);
                }
                const __half2 h = __floats2half2_rn(f[0], f[1]);
                o[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
            }
            reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
            reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
        };
#pragma unroll
        for (int v = tid; v < 2 * KV8_PAGE * (HS / 16); v += 256) {          // pieces of 16 codes: the keys', then the values'
            const bool is_k = v < KV8_PAGE * (HS / 16);
            const int piece = v % (KV8_PAGE * (HS / 16));
            const size_t line = ((size_t)page * kv + kvh) * KV8_PAGE + piece / (HS / 16), at = line * HS + piece % (HS / 16) * 16;
            const uint4 codes = *reinterpret_cast<const uint4*>((is_k ? x.a.c.k : x.a.c.v) + at);
            float ks = x.a.c.k_scale[line], vs = x.a.c.v_scale[line];
            if (!(fabsf(ks) < INFINITY) || !(fabsf(vs) < INFINITY)) { ks = __uint_as_float(0x7fffffffu); vs = 0.f; }
            widen(codes, is_k ? ks : vs, (is_k ? x.k16 : x.v16) + at);
        }
    }
}

// what both entry points refuse
static int kv8_att_args(const char* who, const float* q, long long ldq, int n_heads, const int* pos, const int* slot, const int* block_table, int M, int n_slots, int max_pages, const DlKv8Cache* cache, uint8_t* xq_out, uint8_t* xh_out,
                        int out_mcap, void* y_out, long long ldy, int y_type, Kv8AttArgs* a) {
    const Kv8Rows rows = {pos, slot, block_table, M, n_slots, max_pages, cache ? cache->n_pages : 0};
    if (const int rc = kv8_check(who, cache, &rows)) return rc;
    const int hs = cache->head_size, kv = cache->n_kv_heads;
    if (n_heads < kv || n_heads % kv != 0 || n_heads / kv > 16) { dl_set_error("%s: unsupported head grouping %d/%d", who, n_heads, kv); return -1; }
    if (q == nullptr || (xq_out == nullptr && xh_out == nullptr && y_out == nullptr)) { dl_set_error("%s: no queries or no output", who); return -1; }
    if (ldq < (long long)n_heads * hs || (y_out != nullptr && ldy < (long long)n_heads * hs)) { dl_set_error("%s: rows overlap (ld %lld, %lld)", who, ldq, ldy); return -1; }
    if (y_type != DL_KV8_F32 && y_type != DL_KV8_BF16 && y_type != DL_KV8_F16) { dl_set_error("%s: unsupported output type %d", who, y_type); return -1; }
    if ((xq_out != nullptr || xh_out != nullptr) && ((long long)n_heads * hs % 128 != 0 || out_mcap < M || (xh_out != nullptr && out_mcap % 8 != 0))) {
        dl_set_error("%s: slabs of %d rows, %d columns", who, out_mcap, n_heads * hs);
        return -1;
    }
    *a = {q, ldq, rows, *cache, n_heads, nullptr, nullptr, 0, xq_out, xh_out, out_mcap, y_out, ldy, y_type,
          ((uintptr_t)y_out & (y_type == DL_KV8_F32 ? 15 : 7)) == 0 && ldy % 4 == 0};
    if (M > 65535) { dl_set_error("%s: %d rows (65535 at most)", who, M); return -1; }
    return 0;
}

extern "C" int dl_kv8_attention(const float* q, long long ldq, int n_heads, const int* pos, const int* slot, const int* block_table, int M, int n_slots, int max_pages, const DlKv8Cache* cache, int n_splits, void* scratch, uint8_t* xq_out,
                                uint8_t* xh_out, int out_mcap, void* y_out, long long ldy, int y_type, const int* row_skip, int pdl, void* stream) {
    Kv8AttArgs a;
    if (const int rc = kv8_att_args("dl_kv8_attention", q, ldq, n_heads, pos, slot, block_table, M, n_slots, max_pages, cache, xq_out, xh_out, out_mcap, y_out, ldy, y_type, &a)) return rc;
    if (n_splits > 1 && (scratch == nullptr || ((uintptr_t)scratch & 15) != 0)) { dl_set_error("dl_kv8_attention: n_splits>1 needs scratch, aligned to 16 bytes"); return -1; }
    if (M == 0) return 0;
    if (n_splits > 64) { dl_set_error("dl_kv8_attention: %d splits (64 at most)", n_splits); return -1; }
    if (n_splits < 1) n_splits = 1;
    a.row_skip = row_skip;
    const int hs = cache->head_size;
    return hs == 128 ? ka_decode<128>(a, n_splits, scratch, pdl, stream) : hs == 64 ? ka_decode<64>(a, n_splits, scratch, pdl, stream) : ka_decode<32>(a, n_splits, scratch, pdl, stream);
}

// Rows times heads above which a prompt takes the tcgen05 kernel on widened pages, where there is a workspace.  By rows alone, as positions are on the device: right for
// contexts of up to some 2000 tokens; far behind a conversation fewer rows would gain, too.  us on mma.sync / widened, 32 heads of 128:
//   rows        behind 0     1000         2000         8000         16000
//    16         8.1 / 13.4   11.7 / 20.5  13.8 / 33.1  28.6 / 54.3  47.7 / 78.3
//    64         9.1 / 14.4   14.7 / 22.4  19.4 / 33.5  47.5 / 53.2  85.5 / 79.1
//   128         8.5 / 14.3   18.5 / 22.9  27.8 / 33.9  85.1 / 55.4  162 / 79.1
// 256 behind 2000 55.2 / 35.6, 512 behind 4000 184 / 55.3; 8 heads: 512 behind none 12 / 17, 1024 28.4 / 21.5.  Heads of 64, 32 of them: 128 behind 1000 17.1 / 20.2, 200
// 20.6 / 21.5, 128 behind 8000 84 / 38.7, 256 behind 2000 34.7 / 27.3, 512 behind 4000 102 / 46.7, 4001 behind none 376 / 107; 8 heads: 520 behind none 10.1 / 15, 1024 18.6 / 18.7
static bool ka_widens(long long rows, int n_heads, int hs) { return (hs == 128 && rows * n_heads > 4096) || (hs == 64 && rows * n_heads > 7168); }

extern int dl_attention_prefill_tc_typed(const float* q, int M, int n_heads, int n_kv_heads, int head_size, const void* k_cache, const void* v_cache, const int* pos,
                                         const int* slot, const int* block_table, int max_pages, int page_size, const int* meta, uint8_t* xq_out, uint8_t* xh_out,
                                         int out_mcap, void* y_out, int y_type, bool codes, const PtShares* shares, int n_cache_pages, int pdl, void* stream);
extern int pt_share_ctas();

#define KV8_META_BYTES 128             // of a workspace's scratch: the segments of the launch, then its shares
extern "C" long long dl_kv8_prefill_scratch_bytes(int head_size) {
    return KV8_META_BYTES + pt_share_bytes(head_size);
}

extern "C" int dl_kv8_attention_prefill(const float* q, long long ldq, int n_heads, const int* pos, const int* slot, const int* block_table, int M, int n_slots, int max_pages, const int* meta, int max_seg, const DlKv8Cache* cache, void* k16, void* v16,
                                        void* scratch16, uint8_t* xq_out, uint8_t* xh_out, int out_mcap, void* y_out, long long ldy, int y_type, int pdl, void* stream) {
    const char* who = "dl_kv8_attention_prefill";
    Kv8AttArgs a;
    if (const int rc = kv8_att_args(who, q, ldq, n_heads, pos, slot, block_table, M, n_slots, max_pages, cache, xq_out, xh_out, out_mcap, y_out, ldy, y_type, &a)) return rc;
    if (meta == nullptr || max_seg < 1 || (k16 == nullptr) != (v16 == nullptr) || (k16 == nullptr) != (scratch16 == nullptr)) { dl_set_error("dl_kv8_attention_prefill: a null pointer, or no place for a segment"); return -1; }
    if (M == 0) return 0;
    a.meta = meta;
    a.n_seg = max_seg < 8 ? max_seg : 8;
    const int hs = cache->head_size;
    // (that kernel takes rows side by side, aligned)
    const bool dense = ldq == (long long)n_heads * hs && ((uintptr_t)q & 15) == 0 && (y_out == nullptr || (ldy == ldq && ((uintptr_t)y_out & 15) == 0));
    if (k16 != nullptr && dense && ka_widens(M, n_heads, hs)) {
        if ((((uintptr_t)k16 | (uintptr_t)v16 | (uintptr_t)scratch16) & 15) != 0) { dl_set_error("dl_kv8_attention_prefill: the workspace has to be aligned to 16 bytes"); return -1; }
        uint8_t* scratch = reinterpret_cast<uint8_t*>(scratch16);
        int* meta16 = reinterpret_cast<int*>(scratch);
        const Kv8ExpandArgs x = {a, (__half*)k16, (__half*)v16, meta16};
        static SmemLimit none;
        // a CTA for a page and head, as far as the tables hold them, and eight an SM (four: 130 rows of 32 heads behind 8000 tokens 66 us for 64, 512 behind 16000 156 for 153.5)
        const long long pages = (long long)cache->n_kv_heads * max_pages * min(n_slots, a.n_seg), most = 8 * dl_device_sm_count();
        const dim3 grid((unsigned)(pages < most ? pages : most));
        if (const int rc = hs == 128 ? ka_launch(who, kv8_expand_kernel<128>, none, grid, 1, 256, 0, pdl, stream, x) : ka_launch(who, kv8_expand_kernel<64>, none, grid, 1, 256, 0, pdl, stream, x)) return rc;
        // items that leave half of the SMs without one go to several CTAs each, where the tables may hold sequences that are long enough (PT_SHARE_TOKENS; 500 rows of 32
        // heads of 64 behind none 16.0 us, 17.4 by the instance that looks for shares)
        const int tiles = (M + 127) / 128, items = n_heads / cache->n_kv_heads % 2 == 0 ? tiles * (n_heads / 2) : (tiles + 1) / 2 * n_heads;
        PtShares part = {};
        if (2 * items <= pt_share_ctas() && max_pages >= PT_SHARE_TOKENS / KV8_PAGE) {
            part.arrived = reinterpret_cast<unsigned*>(scratch + KV8_META_BYTES);
            part.norms = reinterpret_cast<float2*>(part.arrived + PT_SHARE_SLOTS * PT_SHARE_WARPS);
            part.sums = reinterpret_cast<float4*>(part.norms + PT_SHARE_SLOTS * PT_SHARE_WARPS * 32);
        }
        return dl_attention_prefill_tc_typed(q, M, n_heads, cache->n_kv_heads, hs, k16, v16, pos, slot, block_table, max_pages, KV8_PAGE, meta16, xq_out, xh_out,
                                             out_mcap, y_out, y_type, true, part.arrived != nullptr ? &part : nullptr, cache->n_pages, 1, stream);
    }
    return hs == 128 ? ka_prompt<128>(a, pdl, stream) : hs == 64 ? ka_prompt<64>(a, pdl, stream) : ka_prompt<32>(a, pdl, stream);
}
