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
#include "smem_limit.cuh"

extern void dl_set_error(const char* fmt, ...);
extern int dl_device_sm_count();
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

// ------------------------------------------------------------------------------------------------
// Both products on mma.sync m16n8k32 with int8 operands: keys and values go in as they lie in the cache, nothing is widened, and sums are exact 32-bit
// integers.  What is f32 is taken as digits of base 256 in rows of the MMA's A operand:
//   a query   n = rint(q 8355000 / max|q|), three signed digits of a head in rows g, g + 8, g + 4 (24 bits of the head's largest value)
//   a weight  n = rint(p s_v 2^(22 - e)), three unsigned digits; e: exponent of the largest p s_v that the row has met (held like a softmax maximum: what
//             was summed is rescaled when it moves), s_v the value's scale.  So each weight is off by 2^-23 of the largest one at most
// Four heads fill the 16 rows.  PROMPT: two digits (16 bits of a query, 15 of a weight), eight (row, head) pairs of one key/value head fill them; four warps
// share a tile's pages.
//
// A warp takes a page (32 tokens) at a time through a private ring of cp.async stages, 16-byte pieces XOR-swizzled by the token so that both ldmatrix
// forms are free of conflicts: no barrier between warps until the final merge.
// ------------------------------------------------------------------------------------------------
#define KA_WARPS 4
#define KA_MIN_SPLIT_PAGES 24        // contexts up to 768 tokens: no split
#define KA_COUNTER_BYTES 65536       // completion counters at scratch offset 0 (dl_attention_scratch_bytes)

DL_DEVINL void ka_cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
DL_DEVINL void ka_ldm(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// two 16 x 16 byte matrices, transposed: lane l gets rows 4 (l % 4) .. + 3 of columns l / 4 and l / 4 + 8 of the first, then of the second
DL_DEVINL void ka_ldm_bytes(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <bool U8> DL_DEVINL void ka_mma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
    if (first) {
        if (U8) asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
        else asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
    } else {
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};" : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
DL_DEVINL float ka_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
DL_DEVINL float ka_max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// shift of a token's 16-byte pieces: eight tokens in a row, and the eight that a phase of the byte-wise ldmatrix reads (two, then the two 8 further on, ...),
// come to lie in eight different columns of 16 bytes
template <int HS> DL_DEVINL int ka_swizzle(int t) {
    const int f = (t & 3) | ((((t >> 2) ^ (t >> 3)) & 1) << 2);
    return HS == 128 ? f : HS == 64 ? f >> 1 : f >> 2;
}

struct Kv8Work {               // what the launch adds to the arguments
    int n_splits, groups;      // groups: CTAs that share a key/value head's query heads
    unsigned* counters;
    float* part_o;             // [M][heads][n_splits][HS]
    float* part_ml;            // [M][heads][n_splits][2]
};

template <int HS, int MT, bool PROMPT, int ST>
__global__ void __launch_bounds__(KA_WARPS * 32) kv8_attention_kernel(const __grid_constant__ Kv8AttArgs a, const __grid_constant__ Kv8Work wk) {
    constexpr int CH = HS / 16, KS = HS / 32, NT = HS / 8;
    constexpr int CODES = KV8_PAGE * HS, STAGE = 2 * CODES + 2 * KV8_PAGE * 4;
    constexpr int SPT = PROMPT ? 8 : 4, SR = MT * SPT;                     // stacked rows of an MMA, of the CTA
    constexpr int TOP = PROMPT ? 14 : 22;                                  // a weight's integer is below 2^(TOP + 1)
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, qd = lane & 3;
    const int kvh = blockIdx.y / wk.groups;
    const int G = a.heads / a.c.n_kv_heads;
    pdl_launch_dependents();
    pdl_wait();

    // which rows and heads: m0 the first row, p0 its position; stacked row s is head h_lo + s (decode), or pair s_lo + s = row * G + head of the group
    int m0, slot, T, h_lo = 0, s_lo = 0, n_live, sp = 0, n_eff = 1, p0 = 0;
    bool bad;
    if constexpr (PROMPT) {
        int tile = gridDim.x - 1 - blockIdx.x, begin = 0, end = 0, i = 0;  // late tiles (long histories) first
        const int n_seg = min(a.meta[0], 8);
        for (; i < n_seg; i++) {
            begin = a.meta[1 + 2 * i];
            end = a.meta[2 + 2 * i];
            if (begin < 0 || end > a.rows.M || end <= begin) continue;
            const int nt = ((end - begin) * G + SR - 1) / SR;
            if (tile < nt) break;
            tile -= nt;
        }
        if (i >= n_seg) return;
        m0 = begin;
        s_lo = tile * SR;
        n_live = min(SR, (end - begin) * G - s_lo);
        p0 = a.rows.pos[begin];
        slot = a.rows.slot[begin];
        bad = p0 >= 0 && (p0 > 0x7fffffff - (end - begin) || kv8_tokens(a.rows, p0 + (end - begin) - 1, slot) < 0);
        T = bad || p0 < 0 ? 0 : p0 + (s_lo + n_live - 1) / G + 1;
    } else {
        m0 = blockIdx.z;
        if (a.row_skip != nullptr && a.row_skip[m0] != 0) return;
        sp = blockIdx.x;
        slot = a.rows.slot[m0];
        T = kv8_tokens(a.rows, a.rows.pos[m0], slot);
        bad = T < 0;
        T = max(T, 0);
        const int per = (G + wk.groups - 1) / wk.groups;
        h_lo = (blockIdx.y % wk.groups) * per;
        n_live = min(per, G - h_lo);
    }
    const int n_pages = (T + KV8_PAGE - 1) / KV8_PAGE;
    if (!PROMPT) {
        n_eff = n_pages <= KA_MIN_SPLIT_PAGES ? 1 : min(wk.n_splits, (n_pages + 7) / 8);
        if (sp >= n_eff) return;
    }
    const int pps = (n_pages + n_eff - 1) / n_eff, pg0 = sp * pps, pg1 = min(n_pages, pg0 + pps);
    const int n_my = max(0, (pg1 - pg0 - warp + KA_WARPS - 1) / KA_WARPS);             // this warp's pages: pg0 + warp + 4 i
    const int* bt = a.rows.block_table + (size_t)(bad ? 0 : slot) * a.rows.max_pages;
    auto row_of = [&](int s) { return PROMPT ? m0 + (s_lo + s) / G : m0; };
    auto head_of = [&](int s) { return kvh * G + (PROMPT ? (s_lo + s) % G : h_lo + s); };

    const uint32_t ring = smem_u32(smem) + warp * (ST * STAGE);
    auto page_at = [&](int i) {
        int p = i < n_my ? bt[pg0 + warp + KA_WARPS * i] : 0;
        if ((unsigned)p >= (unsigned)a.rows.n_pages) { bad = true; p = 0; }
        return p;
    };
    int my_page = page_at(lane);                               // the lanes hold the next 32 page numbers
    auto load = [&](int st, int page) {
        const size_t line = ((size_t)page * a.c.n_kv_heads + kvh) * KV8_PAGE;
        const uint32_t dst = ring + st * STAGE;
        const int8_t* ks = a.c.k + line * HS + lane * 16;
        const int8_t* vs = a.c.v + line * HS + lane * 16;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int idx = j * 32 + lane, t = idx / CH, c = idx % CH;
            const uint32_t d = dst + t * HS + ((c ^ ka_swizzle<HS>(t)) << 4);
            ka_cp16(d, ks + j * 512);
            ka_cp16(d + CODES, vs + j * 512);
        }
        if (lane < 16) ka_cp16(dst + 2 * CODES + lane * 16, (lane < 8 ? a.c.k_scale : a.c.v_scale) + line + (lane & 7) * 4);
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) {
        const int page = __shfl_sync(0xffffffffu, my_page, i);
        if (i < n_my) load(i, page);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // queries: digits in the A fragments; fl: what an integer sum is multiplied with, log2(e) / sqrt(HS) in it
    const bool lower = PROMPT || g < 4;
    uint32_t qf[MT][KS][4];
    float fl[MT];
    int lim[MT];                                               // tokens that the lane's stacked row sees
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int s = mt * SPT + (PROMPT ? g : g & 3);
        const bool live = s < n_live;
        lim[mt] = !live ? 0 : PROMPT ? max(0, min(T, p0 + (s_lo + s) / G + 1)) : T;
        const float* q = a.q + (size_t)row_of(live ? s : 0) * a.ldq + head_of(live ? s : 0) * HS + qd * 4;
        float x[2 * KS][4];
        unsigned top = 0;
        const bool vec = ((uintptr_t)a.q & 15) == 0 && (a.ldq & 3) == 0;
#pragma unroll
        for (int k = 0; k < 2 * KS; k++) {
            if (vec) {
                const float4 v = *reinterpret_cast<const float4*>(q + k * 16);
                x[k][0] = v.x; x[k][1] = v.y; x[k][2] = v.z; x[k][3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) x[k][e] = q[k * 16 + e];
            }
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (queries below 2^-100: their scores are zeros)
        const bool finite = top < 0x7f800000u, zero = !finite || __uint_as_float(top) < KV8_TINY || !live;
        constexpr float MOST = PROMPT ? 32600.f : 8355000.f;
        const float up = zero ? 0.f : MOST / __uint_as_float(top);
        fl[mt] = !finite && live ? __uint_as_float(0x7fffffffu) : zero ? 0.f : __uint_as_float(top) / MOST * (rsqrtf((float)HS) * 1.44269504088896341f) * (PROMPT ? 1.f : lower ? 256.f : 1.f / 256.f);
#pragma unroll
        for (int k = 0; k < 2 * KS; k++) {
            uint32_t n[4];
#pragma unroll
            for (int e = 0; e < 4; e++) n[e] = (uint32_t)(zero ? 0 : __float2int_rn(x[k][e] * up));
            // signed digits: bytes of n + 0x80...80, each less 0x80
#pragma unroll
            for (int e = 0; e < 4; e++) n[e] = PROMPT ? (n[e] + 0x8080u) ^ 0x8080u : (n[e] + 0x808080u) ^ 0x808080u;
            const uint32_t sel = PROMPT ? 0x4051u : lower ? 0x5162u : 0x5140u;
            const uint32_t u = __byte_perm(n[0], n[1], sel), v = __byte_perm(n[2], n[3], sel);
            qf[mt][k / 2][(k & 1) * 2] = __byte_perm(u, v, 0x5410);
            qf[mt][k / 2][(k & 1) * 2 + 1] = lower ? __byte_perm(u, v, 0x7632) : 0u;
        }
    }

    float o[MT][NT][2];
    float run_m[MT], run_l[MT], run_w[MT];                     // maximum of scores, sum of weights (this lane's tokens), largest weight * scale
    int ex[MT];                                                // exponent field of run_w: the unit of o
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        run_m[mt] = -INFINITY;
        run_l[mt] = run_w[mt] = 0.f;
        ex[mt] = 24;
#pragma unroll
        for (int n = 0; n < NT; n++) o[mt][n][0] = o[mt][n][1] = 0.f;
    }
    int all = T;                                               // tokens that every live row of the CTA sees
    if (PROMPT) all = min(T, p0 + s_lo / G + 1);

    // lane's rows of the two ldmatrix forms: tokens and the pieces that they start from
    const int kt = ((lane >> 4) << 3) + (lane & 7), kc = (lane >> 3) & 1;                                   // + 16 j / 2: n-tiles j, j + 1
    const int vr = lane & 15, vt = ((lane >> 4) << 4) + ((vr & 2) << 2) + ((vr >> 2) << 1) + (vr & 1);      // k index 4 a + i is token 8 (i / 2) + 2 a + i % 2
    const uint32_t v_at = vt * HS, v_sw = ka_swizzle<HS>(vt);

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
        const float* scales = reinterpret_cast<const float*>(smem + (size_t)warp * ST * STAGE + st * STAGE + 2 * CODES);
        const int tok0 = (pg0 + warp + KA_WARPS * i) * KV8_PAGE;
        int c[MT][4][4];
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const int t = kt + j * 8;
            const uint32_t base = kb + t * HS, sw = ka_swizzle<HS>(t);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t b[4];
                ka_ldm(b, base + (((2 * k + kc) ^ sw) << 4));
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    ka_mma<false>(c[mt][j], qf[mt][k], b[0], b[1], k == 0);
                    ka_mma<false>(c[mt][j + 1], qf[mt][k], b[2], b[3], k == 0);
                }
            }
        }
        float2 sk[4], sv[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sk[j] = *reinterpret_cast<const float2*>(scales + j * 8 + qd * 2);
            sv[j] = *reinterpret_cast<const float2*>(scales + KV8_PAGE + j * 8 + qd * 2);
        }
        const bool part = tok0 + KV8_PAGE > all;
        uint32_t pa[MT][4];
        float f[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float s[8], w[8], mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int j = e >> 1;
                s[e] = (float)(c[mt][j][e & 1] * 256 + c[mt][j][(e & 1) + 2]) * fl[mt];
                if (!PROMPT) s[e] += __shfl_xor_sync(0xffffffffu, s[e], 16);
                s[e] *= (e & 1) ? sk[j].y : sk[j].x;
                w[e] = (e & 1) ? sv[j].y : sv[j].x;
            }
            if (part) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (tok0 + (e >> 1) * 8 + qd * 2 + (e & 1) >= lim[mt]) { s[e] = -INFINITY; w[e] = 0.f; }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(run_m[mt], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
            const float corr = ka_exp2(run_m[mt] - m_use);
            run_m[mt] = m_new;
            float sum = 0.f, big = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = ka_exp2(s[e] - m_use);
                sum += p;
                w[e] *= p;
                big = ka_max_nan(big, w[e]);
            }
            run_l[mt] = fmaf(run_l[mt], corr, sum);
            big = ka_max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = ka_max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
            big = ka_max_nan(big, run_w[mt] * corr);
            run_w[mt] = big;
            const int e_new = min(max((int)(__float_as_uint(big) >> 23), 24), 254);
            const float up = __uint_as_float((uint32_t)(TOP + 254 - e_new) << 23);
            f[mt] = corr * __uint_as_float((uint32_t)(ex[mt] - TOP) << 23) * up;
            if (big != big) f[mt] = big;
            ex[mt] = e_new;
            uint32_t n[8];
#pragma unroll
            for (int e = 0; e < 8; e++) n[e] = __float_as_uint(fmaf(w[e], up, 8388608.f));     // the integer in the low 23 bits (and 2^23 itself as its top byte)
            const uint32_t sel = PROMPT ? 0x4051u : lower ? 0x5162u : 0x5140u;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t x = __byte_perm(n[4 * u], n[4 * u + 1], sel), y = __byte_perm(n[4 * u + 2], n[4 * u + 3], sel);
                pa[mt][2 * u] = __byte_perm(x, y, 0x5410);
                pa[mt][2 * u + 1] = lower ? __byte_perm(x, y, 0x7632) : 0u;
            }
        }
#pragma unroll
        for (int ch = 0; ch < CH; ch++) {
            uint32_t b[4];
            ka_ldm_bytes(b, vb + v_at + ((ch ^ v_sw) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                int x[4], y[4];
                ka_mma<true>(x, pa[mt], b[0], b[2], true);
                ka_mma<true>(y, pa[mt], b[1], b[3], true);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    o[mt][2 * ch][e] = fmaf(o[mt][2 * ch][e], f[mt], (float)(x[e] * 256 + x[e + 2]));
                    o[mt][2 * ch + 1][e] = fmaf(o[mt][2 * ch + 1][e], f[mt], (float)(y[e] * 256 + y[e + 2]));
                }
            }
        }
        __syncwarp();
        st = st == ST - 1 ? 0 : st + 1;
    }
    bad = __any_sync(0xffffffffu, bad);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                           // the ring is done with
    float* w_acc = reinterpret_cast<float*>(smem);             // [WARPS][SR][HS]
    float* w_ml = w_acc + KA_WARPS * SR * HS;                  // [WARPS][SR][2]
    int* s_last = reinterpret_cast<int*>(w_ml + KA_WARPS * SR * 2);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        run_l[mt] += __shfl_xor_sync(0xffffffffu, run_l[mt], 1);
        run_l[mt] += __shfl_xor_sync(0xffffffffu, run_l[mt], 2);
        if (bad) run_l[mt] = __uint_as_float(0x7fffffffu);
        const float unit = __uint_as_float((uint32_t)(ex[mt] - TOP) << 23) * (PROMPT ? 1.f : lower ? 256.f : 1.f / 256.f);
        const int s = mt * SPT + (PROMPT ? g : g & 3);
        float* w = w_acc + (warp * SR + s) * HS + qd * 2;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                v[e] = o[mt][n][e] * unit;
                if (!PROMPT) v[e] += __shfl_xor_sync(0xffffffffu, v[e], 16);
            }
            if (lower) *reinterpret_cast<float2*>(w + n * 8) = make_float2(v[0], v[1]);
        }
        if (lower && qd == 0) { w_ml[(warp * SR + s) * 2] = run_m[mt]; w_ml[(warp * SR + s) * 2 + 1] = run_l[mt]; }
    }
    __syncthreads();

    // the four warps' shares: a warp takes 32 dimensions of a stacked row at a time (maxima are in units of log2)
    const bool single = n_eff == 1;
    for (int idx = tid; idx < n_live * HS; idx += KA_WARPS * 32) {
        const int s = idx / HS, d = idx % HS;
        float Mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) Mx = fmaxf(Mx, w_ml[(w * SR + s) * 2]);
        const float Mu = Mx == -INFINITY ? 0.f : Mx;
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) {
            const float e = ka_exp2(w_ml[(w * SR + s) * 2] - Mu);
            L += w_ml[(w * SR + s) * 2 + 1] * e;
            O += w_acc[(w * SR + s) * HS + d] * e;
        }
        const int m = row_of(s), hd = head_of(s);
        if (single) {
            const float y = L == 0.f ? 0.f : O / L;
            kv8_store_y(a, m, hd * HS + d, y);
            if (a.xq_out != nullptr || a.xh_out != nullptr) q80_block_store(y, lane, m, (hd * HS + d) >> 5, a.out_mcap, a.xq_out, a.xh_out);
        } else {
            const size_t pidx = ((size_t)m * a.heads + hd) * wk.n_splits + sp;
            wk.part_o[pidx * HS + d] = O;
            if (d == 0) { wk.part_ml[pidx * 2] = Mx; wk.part_ml[pidx * 2 + 1] = L; }
        }
    }
    if (PROMPT || single) return;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        unsigned* counter = &wk.counters[m0 * gridDim.y + blockIdx.y];
        const unsigned prev = atomicAdd(counter, 1u);
        *s_last = prev == (unsigned)n_eff - 1u ? 1 : 0;
        if (*s_last) *counter = 0u;
    }
    __syncthreads();
    if (!*s_last) return;
    __threadfence();
    // a warp merges a head: lane s holds split s's (max, sum), every lane sums its dims over the splits in their order
    for (int s = warp; s < n_live; s += KA_WARPS) {
        constexpr int DPL = HS / 32;
        const int hd = head_of(s);
        const size_t base = ((size_t)m0 * a.heads + hd) * wk.n_splits;
        float ms = -INFINITY, ls = 0.f;
        if (lane < n_eff) { ms = __ldcg(&wk.part_ml[(base + lane) * 2]); ls = __ldcg(&wk.part_ml[(base + lane) * 2 + 1]); }
        const float Mx = warp_max(ms), Mu = Mx == -INFINITY ? 0.f : Mx;
        const float e = lane < n_eff ? ka_exp2(ms - Mu) : 0.f;
        const float L = warp_sum(ls * e);
        float O[DPL];
#pragma unroll
        for (int d = 0; d < DPL; d++) O[d] = 0.f;
#pragma unroll 4
        for (int z = 0; z < n_eff; z++) {
            const float ez = __shfl_sync(0xffffffffu, e, z);
#pragma unroll
            for (int d = 0; d < DPL; d++) O[d] += __ldcg(&wk.part_o[(base + z) * HS + d * 32 + lane]) * ez;
        }
#pragma unroll
        for (int d = 0; d < DPL; d++) {                        // 32 dims at a time: one Q80 block
            const float y = L == 0.f ? 0.f : O[d] / L;
            kv8_store_y(a, m0, hd * HS + d * 32 + lane, y);
            if (a.xq_out != nullptr || a.xh_out != nullptr) q80_block_store(y, lane, m0, hd * DPL + d, a.out_mcap, a.xq_out, a.xh_out);
        }
    }
}

template <int HS, int MT, bool PROMPT, int ST>
static int ka_launch(const char* who, const Kv8AttArgs& a, const Kv8Work& wk, dim3 grid, int pdl, void* stream) {
    constexpr int SR = MT * (PROMPT ? 8 : 4), STAGE = 2 * KV8_PAGE * HS + 2 * KV8_PAGE * 4;
    constexpr int ring = KA_WARPS * ST * STAGE, merge = KA_WARPS * SR * (HS + 2) * 4 + 16, smem = ring > merge ? ring : merge;
    static SmemLimit given;
    if (const int rc = dl_smem_limit(who, kv8_attention_kernel<HS, MT, PROMPT, ST>, smem, given)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(KA_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    if (pdl) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_attention_kernel<HS, MT, PROMPT, ST>, a, wk);
    if (e != cudaSuccess) { dl_set_error("%s launch: %s", who, cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

template <int HS>
static int ka_decode(const Kv8AttArgs& a, int n_splits, void* scratch, int pdl, void* stream) {
    const int kv = a.c.n_kv_heads, G = a.heads / kv, M = a.rows.M;
    Kv8Work wk = {n_splits, G > 8 ? 2 : 1, nullptr, nullptr, nullptr};
    if (n_splits > 1) {
        if ((long long)M * kv * wk.groups * 4 > KA_COUNTER_BYTES) { dl_set_error("dl_kv8_attention: M*n_kv_heads too large for splits"); return -1; }
        uint8_t* at = reinterpret_cast<uint8_t*>(scratch);
        wk.counters = reinterpret_cast<unsigned*>(at);
        wk.part_o = reinterpret_cast<float*>(at + KA_COUNTER_BYTES);
        wk.part_ml = reinterpret_cast<float*>(at + KA_COUNTER_BYTES + ((long long)M * a.heads * n_splits * HS * 4 + 255) / 256 * 256);
    }
    const dim3 grid(n_splits, kv * wk.groups, M);
    constexpr int ST = 2;
    if (G <= 4) return ka_launch<HS, 1, false, ST>("dl_kv8_attention", a, wk, grid, pdl, stream);
    return ka_launch<HS, 2, false, ST>("dl_kv8_attention", a, wk, grid, pdl, stream);
}
template <int HS>
static int ka_prompt(const Kv8AttArgs& a, int pdl, void* stream) {
    constexpr int MT = 2;
    const int kv = a.c.n_kv_heads, G = a.heads / kv;
    const Kv8Work wk = {1, 1, nullptr, nullptr, nullptr};
    const long long tiles = ((long long)a.rows.M * G + MT * 8 - 1) / (MT * 8) + 8;        // upper bound of the tiles of all segments
    return ka_launch<HS, MT, true, 2>("dl_kv8_attention_prefill", a, wk, dim3((unsigned)tiles, kv), pdl, stream);
}

// ------------------------------------------------------------------------------------------------
// Long prompt chunks of heads of 128: the segments' pages widened once to fp16 (fp16(code * scale): 2^-12 of a value, the queries of that kernel are rounded alike),
// then the tcgen05 kernel of the fp16 cache on them, under the same page numbers.  Widening inside that kernel would be done again by every CTA that meets a page
// (rows / 128 * heads / 2 of them).  4001 rows: 12 MB in and 16 MB out, beside 131 GFLOP.
//
// A line with a NaN (of the key or the value) becomes a key of NaN and a value of zeros: the rows that see it give NaN, and the weights of 0 that others
// have for it do not.  Values beyond fp16's range saturate.  What that kernel does not look at is looked at here: the segments that are in the tables are listed
// for it, rows of the others get NaN.
// ------------------------------------------------------------------------------------------------
struct Kv8ExpandArgs {
    Kv8AttArgs a;
    __half* k16;               // [pages][kv][32][128]
    __half* v16;
    int* meta_out;             // [17]
};

__global__ void __launch_bounds__(256) kv8_expand_kernel(const __grid_constant__ Kv8ExpandArgs x) {
    constexpr int HS = 128;
    __shared__ int first[9], seg[8][3];                        // items ahead of a segment; begin, end, slot
    __shared__ int ok[8];
    const int tid = threadIdx.x, kv = x.a.c.n_kv_heads;
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) {
        const int n = max(0, min(x.a.meta[0], 8));
        int at = 0;
        for (int i = 0; i < 8; i++) {
            first[i] = at;
            const int b = i < n ? x.a.meta[1 + 2 * i] : 0, e = i < n ? x.a.meta[2 + 2 * i] : 0;
            const bool rows = b >= 0 && e <= x.a.rows.M && e > b;
            const int p = rows ? x.a.rows.pos[b] : 0, s = rows ? x.a.rows.slot[b] : 0;
            ok[i] = rows && p >= 0 && p <= 0x7fffffff - (e - b) && kv8_tokens(x.a.rows, p + (e - b) - 1, s) > 0;
            seg[i][0] = b; seg[i][1] = rows ? e : b; seg[i][2] = s;
            if (ok[i]) at += (p + (e - b) + KV8_PAGE - 1) / KV8_PAGE * kv;
        }
        first[8] = at;
    }
    __syncthreads();
    // pages that are not there: the first CTA, which lists the segments, takes theirs as one that is not in the tables
    for (int i = 0; i < 8; i++) {
        if (!ok[i]) continue;
        const int* bt = x.a.rows.block_table + (size_t)seg[i][2] * x.a.rows.max_pages;
        const int pages = (first[i + 1] - first[i]) / kv;
        bool bad = false;
        if (blockIdx.x == 0)
            for (int p = tid; p < pages; p += 256) bad |= (unsigned)bt[p] >= (unsigned)x.a.rows.n_pages;
        if (__syncthreads_or(bad) && tid == 0) ok[i] = 0;
    }
    __syncthreads();
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
        const size_t line = ((size_t)page * kv + kvh) * KV8_PAGE + (tid >> 3);
        const size_t at = line * HS + (tid & 7) * 16;
        const uint4 kc = *reinterpret_cast<const uint4*>(x.a.c.k + at), vc = *reinterpret_cast<const uint4*>(x.a.c.v + at);
        float ks = x.a.c.k_scale[line], vs = x.a.c.v_scale[line];
        if (!(fabsf(ks) < INFINITY) || !(fabsf(vs) < INFINITY)) { ks = __uint_as_float(0x7fffffffu); vs = 0.f; }
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
        widen(kc, ks, x.k16 + at);
        widen(vc, vs, x.v16 + at);
    }
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
    if (n_splits > 32) { dl_set_error("dl_kv8_attention: %d splits (32 at most)", n_splits); return -1; }
    if (n_splits < 1) n_splits = 1;
    a.row_skip = row_skip;
    const int hs = cache->head_size;
    return hs == 128 ? ka_decode<128>(a, n_splits, scratch, pdl, stream) : hs == 64 ? ka_decode<64>(a, n_splits, scratch, pdl, stream) : ka_decode<32>(a, n_splits, scratch, pdl, stream);
}

// Rows times heads above which heads of 128 take the tcgen05 kernel on widened pages, where there is a workspace (us on mma.sync / widened, 32 heads: 128 rows
// behind 1000 tokens 21 / 24, behind 8000 95 / 92, 256 behind 2000 63 / 36, 512 behind 4000 208 / 60; 8 heads: 512 rows behind none 13.5 / 17.9, 1024 27 / 22)
#define KV8_EXPAND_MIN_WORK 4096

extern int dl_attention_prefill_tc_typed(const float* q, int M, int n_heads, int n_kv_heads, int head_size, const void* k_cache, const void* v_cache, const int* pos,
                                         const int* slot, const int* block_table, int max_pages, int page_size, const int* meta, uint8_t* xq_out, uint8_t* xh_out,
                                         int out_mcap, void* y_out, int y_type, int n_cache_pages, int pdl, void* stream);

extern "C" int dl_kv8_attention_prefill(const float* q, long long ldq, int n_heads, const DlKv8Rows* rows, const int* meta, const DlKv8Cache* cache, void* k16, void* v16,
                                        int* meta16, uint8_t* xq_out, uint8_t* xh_out, int out_mcap, void* y_out, long long ldy, int y_type, int pdl, void* stream) {
    Kv8AttArgs a;
    if (const int rc = kv8_att_args("dl_kv8_attention_prefill", q, ldq, n_heads, rows, cache, xq_out, xh_out, out_mcap, y_out, ldy, y_type, &a)) return rc;
    if (meta == nullptr || (k16 == nullptr) != (v16 == nullptr) || (k16 == nullptr) != (meta16 == nullptr)) { dl_set_error("dl_kv8_attention_prefill: a null pointer"); return -1; }
    if (rows->M == 0) return 0;
    a.meta = meta;
    const int hs = cache->head_size;
    // (that kernel takes rows side by side, aligned)
    const bool dense = ldq == (long long)n_heads * hs && ((uintptr_t)q & 15) == 0 && (y_out == nullptr || (ldy == ldq && ((uintptr_t)y_out & 15) == 0));
    if (k16 != nullptr && hs == 128 && dense && (long long)rows->M * n_heads > KV8_EXPAND_MIN_WORK) {
        if ((((uintptr_t)k16 | (uintptr_t)v16) & 15) != 0) { dl_set_error("dl_kv8_attention_prefill: the workspace has to be aligned to 16 bytes"); return -1; }
        const Kv8ExpandArgs x = {a, (__half*)k16, (__half*)v16, meta16};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(4 * dl_device_sm_count());
        cfg.blockDim = dim3(256);
        cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl ? 1 : 0;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_expand_kernel, x);
        if (e != cudaSuccess) { dl_set_error("dl_kv8_attention_prefill launch: %s", cudaGetErrorString(e)); return -(int)e; }
        return dl_attention_prefill_tc_typed(q, rows->M, n_heads, cache->n_kv_heads, hs, k16, v16, rows->pos, rows->slot, rows->block_table, rows->max_pages, KV8_PAGE, meta16,
                                             xq_out, xh_out, out_mcap, y_out, y_type, cache->n_pages, 1, stream);
    }
    return hs == 128 ? ka_prompt<128>(a, pdl, stream) : hs == 64 ? ka_prompt<64>(a, pdl, stream) : ka_prompt<32>(a, pdl, stream);
}
