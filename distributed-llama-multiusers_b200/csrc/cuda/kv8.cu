// Writing the 8-bit token cache and reading it back (kv8.cuh has the format).
//
// kv8_write: the merged q|k|v rows of a layer in one pass -- rotary positions on queries and keys (pairs of neighbouring values, OP_ROPE_LLAMA,
// ropeLlamaForward_F32_F32: nn-cpu-ops.cpp:1090-1120), keys and values to their pages (OP_SHIFT, shiftForward_F32_F32: nn-cpu-ops.cpp:1253-1275)
// as codes and scales.
//
// A code is a rounding, and an input a hair beside a border lands on either side of it: so that the same rows give the same codes however they are
// computed, keys are turned in 64 bits (angle, sine, cosine and both products) and rounded once to f32, and x * factor goes to the nearest integer in
// one rounding, an fma with 1.5 2^23.  Queries take f32 products of the same sines and cosines.  The sines of a row are formed once for all heads.
//
// What bounds them: few rows, one chain of latencies; many rows read, the bytes; many rows written, still the chains (position, sines in 64 bits and a barrier come ahead of a
// CTA's loads: DRAM is active 45 % of the time).  Written, 32 query heads and 8 key/value heads of 128: one row 3.1 us, 32 3.3, 4001 (172 MB) 37.6, 4.6 TB/s; read as fp16: 4001 rows 8.3 us, 100003 (621 MB) 101.9, 6.1 TB/s, of which a copy reaches 6.45.
#include <type_traits>
#include "epilogue.cuh"
#include "kv8.cuh"

extern void dl_set_error(const char* fmt, ...);
extern int dl_device_sm_count();

struct Kv8WriteArgs {
    const float* qkv;          // [M][ld]: heads | kv heads | kv heads
    long long ld;
    const float* freqs;        // [HS / 2] or NULL: no rotation
    float* q_out;              // [M][ldq]
    long long ldq;
    Kv8Rows rows;
    DlKv8Cache c;
    int heads;
};

#define KV8_WRITE_WARPS 4

template <bool VEC> DL_DEVINL float4 kv8_fetch(const float* src, bool live) {
    if (!live) return make_float4(0.f, 0.f, 0.f, 0.f);
    return VEC ? __ldcs(reinterpret_cast<const float4*>(src)) : make_float4(src[0], src[1], src[2], src[3]);
}

// grid (M, shares of a row's heads).  A warp takes a "unit" of 32 / (HS / 4) heads of one kind at a time, a lane four neighbouring values of the same place in
// every head, so that it reads its sines once a row; six units in flight (4001 rows of 48 heads of 128 37 us, 38.5 with one)
template <int HS, bool VEC>
__global__ void __launch_bounds__(KV8_WRITE_WARPS * 32) kv8_write_kernel(const __grid_constant__ Kv8WriteArgs a) {
    constexpr int LPH = HS / 4, HPW = 32 / LPH, AHEAD = 6;     // lanes a head, heads a unit, units in flight
    __shared__ double2 turn[HS / 2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, li = lane % LPH, hi = lane / LPH;
    const int kv = a.c.n_kv_heads, nq = (a.heads + HPW - 1) / HPW, nk = (kv + HPW - 1) / HPW;
    const int m = blockIdx.x, first = blockIdx.y * KV8_WRITE_WARPS + warp, step = gridDim.y * KV8_WRITE_WARPS;
    pdl_launch_dependents();
    pdl_wait();
    const int pos = a.rows.pos[m], slot = a.rows.slot[m];
    if (kv8_tokens(a.rows, pos, slot) <= 0) return;            // (uniform for the CTA)
    const int named = a.rows.block_table[(size_t)slot * a.rows.max_pages + pos / KV8_PAGE], page = (unsigned)named < (unsigned)a.rows.n_pages ? named : -1;
    if (tid < HS / 2) {
        double s = 0., c = 1.;
        if (a.freqs != nullptr) sincos((double)pos * (double)a.freqs[tid], &s, &c);
        turn[tid] = make_double2(c, s);
    }
    __syncthreads();
    const double2 t0 = turn[2 * li], t1 = turn[2 * li + 1];
    const float c0 = (float)t0.x, s0 = (float)t0.y, c1 = (float)t1.x, s1 = (float)t1.y;
    const float* src = a.qkv + m * a.ld + hi * HS + li * 4;
    float* dst = a.q_out + m * a.ldq + hi * HS + li * 4;
    for (int u0 = first; u0 < nq + 2 * nk; u0 += AHEAD * step) {
        float4 x[AHEAD];
#pragma unroll
        for (int b = 0; b < AHEAD; b++) {
            const int u = u0 + b * step, w = u - nq;       // queries, keys (w < nk), values
            if (u < nq) x[b] = kv8_fetch<VEC>(src + u * (HPW * HS), u * HPW + hi < a.heads);
            else if (w < nk) x[b] = kv8_fetch<VEC>(src + (a.heads + w * HPW) * HS, w * HPW + hi < kv);
            else x[b] = kv8_fetch<VEC>(src + (a.heads + kv + (w - nk) * HPW) * HS, w < 2 * nk && (w - nk) * HPW + hi < kv);
        }
#pragma unroll
        for (int b = 0; b < AHEAD; b++) {
            const int u = u0 + b * step, w = u - nq;
            if (u < nq) {
                if (u * HPW + hi >= a.heads) continue;
                float4 y = x[b];
                if (a.freqs != nullptr) y = make_float4(x[b].x * c0 - x[b].y * s0, x[b].x * s0 + x[b].y * c0, x[b].z * c1 - x[b].w * s1, x[b].z * s1 + x[b].w * c1);
                float* at = dst + u * (HPW * HS);
                if (VEC) *reinterpret_cast<float4*>(at) = y;
                else { at[0] = y.x; at[1] = y.y; at[2] = y.z; at[3] = y.w; }
                continue;
            }
            if (w >= 2 * nk) break;
            const bool is_k = w < nk;
            const int h = (is_k ? w : w - nk) * HPW + hi;
            float k[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
            if (is_k && a.freqs != nullptr) {
                const double x0 = k[0], x1 = k[1], x2 = k[2], x3 = k[3];
                k[0] = (float)(x0 * t0.x - x1 * t0.y);
                k[1] = (float)(x0 * t0.y + x1 * t0.x);
                k[2] = (float)(x2 * t1.x - x3 * t1.y);
                k[3] = (float)(x2 * t1.y + x3 * t1.x);
            }
            // the line's largest magnitude as bits: an infinity or a NaN is above every number
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(k[e]) & 0x7fffffffu);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (h >= kv || page < 0) continue;
            const float amax = __uint_as_float(top);
            float scale = 0.f, factor = 0.f;
            if (top >= 0x7f800000u) scale = __uint_as_float(0x7fffffffu);      // the line reads back as NaN
            else if (amax >= KV8_TINY) { scale = __fdiv_rn(amax, 127.f); factor = __fdiv_rn(127.f, amax); }
            uint32_t code = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) code |= (__float_as_uint(__fmaf_rn(top >= 0x7f800000u ? 0.f : k[e], factor, 12582912.f)) & 0xffu) << (8 * e);
            const size_t line = ((size_t)page * kv + h) * KV8_PAGE + pos % KV8_PAGE;
            reinterpret_cast<uint32_t*>((is_k ? a.c.k : a.c.v) + line * HS)[li] = code;
            if (li == 0) (is_k ? a.c.k_scale : a.c.v_scale)[line] = scale;
        }
    }
}

struct Kv8ReadArgs {
    void* k_out;               // [M][ld]
    void* v_out;
    long long ld;
    Kv8Rows rows;
    DlKv8Cache c;
    int per_cta;               // rows of a CTA
};

template <typename T> DL_DEVINL T kv8_from_float(float x);
template <> DL_DEVINL float kv8_from_float<float>(float x) { return x; }
template <> DL_DEVINL __half kv8_from_float<__half>(float x) { return __float2half_rn(x); }
template <> DL_DEVINL __nv_bfloat16 kv8_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

#define KV8_READ_WARPS 8
#define KV8_READ_ROWS 32       // most rows of a CTA
#define KV8_READ_AHEAD 8       // pieces of a lane in flight (100003 tokens of 8 heads of 128 into fp16: 102 us, 165 with one)

// a warp takes a row at a time, a lane the codes of 16 bytes of output; rows without a token read as zeros, rows that are not in the tables as NaN
template <int HS, typename T, bool VEC>
__global__ void __launch_bounds__(KV8_READ_WARPS * 32) kv8_read_kernel(const __grid_constant__ Kv8ReadArgs a) {
    constexpr int N = 16 / (int)sizeof(T), UPH = HS / N;       // values of a lane, lanes a head
    __shared__ long long at[KV8_READ_ROWS];                    // first line of the row's token (of head 0); -1: none, -2: NaN
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();
    const int m0 = blockIdx.x * a.per_cta, n = min(a.per_cta, a.rows.M - m0), kv = a.c.n_kv_heads;
    if (tid < n) {
        const int pos = a.rows.pos[m0 + tid], slot = a.rows.slot[m0 + tid], t = kv8_tokens(a.rows, pos, slot);
        long long line = t == 0 ? -1 : -2;
        if (t > 0) {
            const int page = a.rows.block_table[(size_t)slot * a.rows.max_pages + pos / KV8_PAGE];
            if ((unsigned)page < (unsigned)a.rows.n_pages) line = (long long)page * kv * KV8_PAGE + pos % KV8_PAGE;
        }
        at[tid] = line;
    }
    __syncthreads();
    const int units = 2 * kv * UPH;
    for (int r = warp; r < n; r += KV8_READ_WARPS) {
        const long long line0 = at[r];
        for (int u0 = lane; u0 < units; u0 += 32 * KV8_READ_AHEAD) {
            uint32_t w[KV8_READ_AHEAD][N / 4];
            float s[KV8_READ_AHEAD];
#pragma unroll
            for (int b = 0; b < KV8_READ_AHEAD; b++) {
                const int u = u0 + b * 32, g = u / UPH;
                const bool is_k = g < kv;
                s[b] = line0 == -1 ? 0.f : __uint_as_float(0x7fffffffu);
#pragma unroll
                for (int e = 0; e < N / 4; e++) w[b][e] = 0;
                if (u >= units || line0 < 0) continue;
                const long long line = line0 + (long long)(is_k ? g : g - kv) * KV8_PAGE;
                s[b] = (is_k ? a.c.k_scale : a.c.v_scale)[line];
                const int8_t* src = (is_k ? a.c.k : a.c.v) + line * HS + u % UPH * N;
                if (N == 8) { const uint2 x = __ldcs(reinterpret_cast<const uint2*>(src)); w[b][0] = x.x; w[b][N / 4 - 1] = x.y; }
                else w[b][0] = __ldcs(reinterpret_cast<const uint32_t*>(src));
            }
#pragma unroll
            for (int b = 0; b < KV8_READ_AHEAD; b++) {
                const int u = u0 + b * 32, g = u / UPH;
                if (u >= units) break;
                const bool is_k = g < kv;
                alignas(16) T o[N];
#pragma unroll
                for (int e = 0; e < N; e++) o[e] = kv8_from_float<T>((float)(int8_t)(w[b][e / 4] >> (8 * (e % 4))) * s[b]);
                T* dst = reinterpret_cast<T*>(is_k ? a.k_out : a.v_out) + (m0 + r) * a.ld + (is_k ? g : g - kv) * HS + u % UPH * N;
                if (VEC) __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<const uint4*>(o));
                else {
#pragma unroll
                    for (int e = 0; e < N; e++) dst[e] = o[e];
                }
            }
        }
    }
}

int kv8_check(const char* who, const DlKv8Cache* c, const Kv8Rows* r) {
    if (c == nullptr) { dl_set_error("%s: no cache", who); return -1; }
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 128) { dl_set_error("%s: unsupported head_size %d (32, 64 or 128)", who, c->head_size); return -1; }
    if (c->n_kv_heads < 1 || c->n_pages < 1) { dl_set_error("%s: %d kv heads, %d pages", who, c->n_kv_heads, c->n_pages); return -1; }
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !r->pos || !r->slot || !r->block_table) { dl_set_error("%s: a null pointer", who); return -1; }
    if ((((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 15) != 0) { dl_set_error("%s: the cache has to be aligned to 16 bytes", who); return -1; }
    if (r->M < 0 || r->n_slots < 1 || r->max_pages < 1 || r->max_pages > 0x7fffffff / KV8_PAGE) { dl_set_error("%s: %d rows, block table [%d][%d]", who, r->M, r->n_slots, r->max_pages); return -1; }
    return 0;
}

template <typename K, typename A>
static int kv8_launch(const char* who, K kernel, const A& a, dim3 grid, int threads, int pdl, void* stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    if (pdl) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) { dl_set_error("%s launch: %s", who, cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

extern "C" int dl_kv8_write(const float* qkv, long long ld_qkv, int n_heads, const float* freqs, const int* pos, const int* slot, const int* block_table, int M, int n_slots, int max_pages, float* q_out, long long ld_q,
                            const DlKv8Cache* cache, int pdl, void* stream) {
    const Kv8Rows rows = {pos, slot, block_table, M, n_slots, max_pages, cache ? cache->n_pages : 0};
    if (const int rc = kv8_check("dl_kv8_write", cache, &rows)) return rc;
    const int hs = cache->head_size, kv = cache->n_kv_heads;
    if (n_heads < 0 || qkv == nullptr || (n_heads > 0 && q_out == nullptr)) { dl_set_error("dl_kv8_write: %d heads, or a null pointer", n_heads); return -1; }
    if (ld_qkv < (long long)(n_heads + 2 * kv) * hs || (n_heads > 0 && ld_q < (long long)n_heads * hs)) { dl_set_error("dl_kv8_write: rows overlap (ld %lld, %lld)", ld_qkv, ld_q); return -1; }
    if (M == 0) return 0;
    // few rows: a row's heads go to as many CTAs as the SMs have room for, a unit for each warp at most
    const int per_warp = 128 / hs, units = (n_heads + per_warp - 1) / per_warp + 2 * ((kv + per_warp - 1) / per_warp), most = (units + KV8_WRITE_WARPS - 1) / KV8_WRITE_WARPS;
    const int share = 4 * dl_device_sm_count() / M;
    Kv8WriteArgs a = {qkv, ld_qkv, freqs, q_out, ld_q, rows, *cache, n_heads};
    const bool vec = ((uintptr_t)qkv & 15) == 0 && ((uintptr_t)q_out & 15) == 0 && ld_qkv % 4 == 0 && (n_heads == 0 || ld_q % 4 == 0);
    const dim3 grid(M, share < 1 ? 1 : share < most ? share : most);
    auto go = [&](auto hs_c) {
        constexpr int HS = decltype(hs_c)::value;
        return vec ? kv8_launch("dl_kv8_write", kv8_write_kernel<HS, true>, a, grid, KV8_WRITE_WARPS * 32, pdl, stream)
                   : kv8_launch("dl_kv8_write", kv8_write_kernel<HS, false>, a, grid, KV8_WRITE_WARPS * 32, pdl, stream);
    };
    if (hs == 128) return go(std::integral_constant<int, 128>());
    if (hs == 64) return go(std::integral_constant<int, 64>());
    return go(std::integral_constant<int, 32>());
}

extern "C" int dl_kv8_read(const int* pos, const int* slot, const int* block_table, int M, int n_slots, int max_pages, const DlKv8Cache* cache, void* k_out, void* v_out, long long ld, int out_type, int pdl, void* stream) {
    const Kv8Rows rows = {pos, slot, block_table, M, n_slots, max_pages, cache ? cache->n_pages : 0};
    if (const int rc = kv8_check("dl_kv8_read", cache, &rows)) return rc;
    const int hs = cache->head_size;
    if (k_out == nullptr || v_out == nullptr) { dl_set_error("dl_kv8_read: a null pointer"); return -1; }
    if (out_type != DL_KV8_F32 && out_type != DL_KV8_BF16 && out_type != DL_KV8_F16) { dl_set_error("dl_kv8_read: unsupported output type %d", out_type); return -1; }
    if (ld < (long long)cache->n_kv_heads * hs) { dl_set_error("dl_kv8_read: rows overlap (ld %lld)", ld); return -1; }
    if (M == 0) return 0;
    const int sms = dl_device_sm_count();
    int per = (M + 8 * sms - 1) / (8 * sms);
    per = per < 1 ? 1 : per > KV8_READ_ROWS ? KV8_READ_ROWS : per;
    Kv8ReadArgs a = {k_out, v_out, ld, rows, *cache, per};
    const int size = out_type == DL_KV8_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 && ld * size % 16 == 0;
    const dim3 grid((M + per - 1) / per);
    auto go = [&](auto hs_c, auto zero) {
        constexpr int HS = decltype(hs_c)::value;
        using T = decltype(zero);
        return vec ? kv8_launch("dl_kv8_read", kv8_read_kernel<HS, T, true>, a, grid, KV8_READ_WARPS * 32, pdl, stream)
                   : kv8_launch("dl_kv8_read", kv8_read_kernel<HS, T, false>, a, grid, KV8_READ_WARPS * 32, pdl, stream);
    };
    auto typed = [&](auto hs_c) {
        if (out_type == DL_KV8_F32) return go(hs_c, float());
        if (out_type == DL_KV8_BF16) return go(hs_c, __nv_bfloat16());
        return go(hs_c, __half());
    };
    if (hs == 128) return typed(std::integral_constant<int, 128>());
    if (hs == 64) return typed(std::integral_constant<int, 64>());
    return typed(std::integral_constant<int, 32>());
}
