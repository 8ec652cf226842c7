// A token for every row of logits from given random numbers: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T); the order of tokens: largest logit first, of equal ones the lowest index first
//   top-k   a token stays if fewer than k are ahead of it;
//   top-p   of those a token stays if the weight ahead of it is below p times the weight of what top-k leaves;
//   min-p   of those a token stays if w_i >= min_p (the largest weight is 1)
//   the token: in the order of the vocabulary the first one where the sum of the weights that stay is above coin times their total
// so what stays is always the front of the order, and one border (logit, index) tells it.  T <= 0: the first of the largest.
//
// A cluster of CTAs reads a row, from memory for its maximum, from the L2 then.  Nothing is sorted: "with which token does a sum, taken in some order, reach a target" is answered by bins and,
// within the bin, of a few tokens, by comparing them with each other (StRow::select).  What takes part in that is a list in the first CTA's shared memory, in which the border has to lie:
//   top-k   The least of as many maxima, each over tokens of its own, as k or more is not above the k-th largest logit.  The first pass leaves such maxima (of threads, of 2, 4, .. 32
//           threads: by steps of 4, of more than one row in a thousand more was left than the list takes); what is not below the least of them, some thousand tokens, goes into the list, and the rest of the row has no part: the first CTA does it all.
//   top-p   A second pass counts the tokens in 4096 bins of their distance to the maximum.  A bin's weights differ by 0.5 %, so that the counts tell the sums to some 0.02 % (of heavy tokens, which
//           would be most of that, their weights count: without it the list was too short for one row in a hundred, 200 rows 347 us instead of 152), and the border to a few bins.  A third pass adds up the weights: of the row, for the target, and of what lies ahead of those bins, for each warp's run of the row; the bins' tokens go into the list.
//           The first CTA finds the border there, and the warp's run in which the token lies.
//   else    as top-p, without a border.
// Where the list does not do -- more tokens than it takes, a border that is not in it -- all CTAs select over the whole row, by bins that are divided until few tokens are left.
//
// Weights are whole numbers of 2^-44, so that sums do not depend on their order; they are off by 2^-29 of themselves (a table of 64 powers of two and a
// polynomial, after P. T. P. Tang's table-driven exponential, on the difference and the factor as pairs of f32 numbers) and half a unit, 2^-45 of the largest one's: a sum over V tokens by 2^-29 of
// itself and V 2^-45 at most, 2^-26 for the largest vocabulary.  With sums of f32 results a coin next to a border between two tokens would fall on the other side once in some thousand rows.
//
// What bounds it: for few rows some 25 phases, one behind the other, each a barrier of the cluster or a chain through shared memory, and code that is read once (one row of 128256 logits, us: top-p 22.6,
// top-k and top-p 16, neither 12, min-p alone 9; the bytes 0.08).  200 rows take 153, 64, 102 and 47 us (the bytes 16): 100, 24, 72 and 15 instructions a token, which alone would take 70, 17, 50 and 11 us.
// With seven warps a scheduler (56 registers) they issue in 54, 37, 57 and 27 % of its cycles; what the warps wait for in the others are loads, of rows that come from the L2 the second time and in part
// from memory (136 to 206 MB for 103), first, then what the instruction ahead has to leave.
#include <math_constants.h>
#include <cuda_bf16.h>
#include "common.cuh"
#include "smem_limit.cuh"

#define ST_BINS 256
#define ST_FINE 4096                   // bins of top-p's counts
#define ST_HEAVY 1024                  // ... of which the first ones' tokens count by their weights
#define ST_LIST 6144
#define ST_LEVELS 6                    // sizes of the groups of threads whose maxima bound top-k
#define ST_FEW 128                     // tokens that are compared with each other
#define ST_MAX_CTAS 16
#define ST_MAX_WARPS 32
#define ST_REACH 20.0f                 // how far below the maximum the bins reach, in units of the exponent (a vocabulary of weights beyond it: 1e-3 of the largest)
#define ST_IDX_BITS 20
#define ST_ONE (1ull << 44)
#define ST_AHEAD 4                     // loads of four logits in flight for each thread

typedef unsigned long long u64;

struct StArgs {
    const void* logits;
    long long ld;
    const float *temperature, *top_p, *min_p, *coin;
    const int* top_k;
    int* tokens;
    float* prob;
    int vocab, slice;
    int wide;                          // four logits of a row can be read at a time
};

struct StSums { u64 weight; u64 count; };

// what the CTAs of a row leave for each other; in each CTA's shared memory
struct alignas(16) StShared {
    union {
        u64 list[ST_LIST];             // keys: this CTA's from the front; in CTA 0's the other ones' from the back
        struct { unsigned fine[ST_FINE], fine_sum[ST_FINE]; } count;      // ahead of it: this CTA's counts, the cluster's
    };
    unsigned hist[4][ST_BINS];         // this CTA's counts, and weights in three parts of 15 bits
    StSums merged[ST_BINS];            // the cluster's bins
    u64 run_sum[ST_MAX_CTAS * ST_MAX_WARPS];      // in CTA 0's: the weights of each warp's run
    u64 few_order[ST_FEW], few_weight[ST_FEW];
    u64 lo[ST_MAX_CTAS], hi[ST_MAX_CTAS];
    u64 cta_sum[ST_MAX_CTAS];
    float top[ST_MAX_CTAS], low[ST_LEVELS][ST_MAX_CTAS];      // each CTA's largest logit; the least of the largest ones of its threads, of 2, 4, .. 32 of them
    StSums above, inside;              // of the bin found: what lies ahead of it and in it
    int bin, bin_from, bin_to;
    unsigned listed, others, few, done, first;      // listed: this CTA's; others: in CTA 0's the other ones'
    u64 found, upto;                   // the order of the token found, the sum up to it
    u64 warp_sum[ST_MAX_WARPS];
    float warp_top[ST_MAX_WARPS], warp_low[ST_LEVELS - 1][ST_MAX_WARPS];
    StSums red[ST_MAX_WARPS];
    uint2 pow2[64];                    // 2^(j / 64): times 2^31, and as f32
};

DL_DEVINL unsigned st_order(float x) {
    const unsigned b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
// logit and index as one number, larger for what is ahead
#define ST_IDX_MASK ((1ull << ST_IDX_BITS) - 1)
DL_DEVINL u64 st_key(float x, int i) { return ((u64)st_order(x + 0.f) << ST_IDX_BITS) | (ST_IDX_MASK - i); }      // (a zero has no sign)
DL_DEVINL float st_logit(u64 key) {
    const unsigned q = (unsigned)(key >> ST_IDX_BITS);
    return __uint_as_float((q & 0x80000000u) ? q ^ 0x80000000u : ~q);
}
DL_DEVINL int st_index(u64 key) { return (int)(ST_IDX_MASK - (key & ST_IDX_MASK)); }

DL_DEVINL u64 st_max_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}
DL_DEVINL u64 st_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct StScale { float m, c_hi, c_lo; };      // maximum of the row, log2(e) / T as two numbers

// round(2^44 exp((x - m) / T)) for x below m, without a branch
DL_DEVINL u64 st_weight_below(float x, const StScale& s, const uint2* pow2) {
    const float d = x - s.m, p = __fmul_rn(d, s.c_hi);          // (not part of a sum: its error is e)
    const float b = d - x, lost = (x - (d - b)) + (-s.m - b);   // x - m = d + lost
    const float e = fmaf(lost, s.c_hi, fmaf(d, s.c_lo, fmaf(d, s.c_hi, -p)));
    const float t = __fadd_rn(p, 196608.f);                              // 1.5 2^17: p to the nearest 1 / 64
    const int k = __float_as_int(t) - __float_as_int(196608.f);
    const float r = __fadd_rn(__fsub_rn(p, t - 196608.f), e);                   // at most 2^-7
    const float q = r * fmaf(r, fmaf(r, fmaf(r, 0.00961812911f, 0.0555041087f), 0.240226507f), 0.693147181f);      // 2^r - 1
    const uint2 f = pow2[k & 63];
    const int low = __float_as_int(fmaf(__uint_as_float(f.y), q, 0.046875f)) - __float_as_int(0.046875f);        // 1.5 2^-5: units of 2^-28
    const u64 w = (u64)(f.x + ((unsigned)low << 3)) << 14;
    return p > -46.f ? ((w >> (-(k >> 6) & 63)) + 1) >> 1 : 0;      // (not: an infinite difference, whose steps are no numbers)
}
DL_DEVINL u64 st_weight(float x, const StScale& s, const uint2* pow2) { return x == s.m ? ST_ONE : st_weight_below(x, s, pow2); }      // (infinities among the former)

// u f rounded down, and whether something was lost; f in [0, 1)
DL_DEVINL u64 st_times(u64 u, float f, bool& more) {
    const u64 scaled = (u64)((double)f * 9223372036854775808.0) << 1;      // 2^64 f (24 bits of it; below 2^-40 some are lost)
    more = u * scaled != 0;
    return __umul64hi(u, scaled);
}

template <typename T> DL_DEVINL float4 st_load4(const T* p, bool wide);
template <> DL_DEVINL float4 st_load4<float>(const float* p, bool wide) {
    if (wide) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
template <> DL_DEVINL float4 st_load4<__nv_bfloat16>(const __nv_bfloat16* p, bool wide) {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
    uint2 r;
    if (wide) r = *reinterpret_cast<const uint2*>(p);
    else r = make_uint2(q[0] | (unsigned)q[1] << 16, q[2] | (unsigned)q[3] << 16);
    return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u));
}
template <> DL_DEVINL float4 st_load4<__half>(const __half* p, bool wide) {
    if (!wide) return make_float4(__half2float(p[0]), __half2float(p[1]), __half2float(p[2]), __half2float(p[3]));
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <typename T> DL_DEVINL float st_load1(const T* p);
template <> DL_DEVINL float st_load1<float>(const float* p) { return *p; }
template <> DL_DEVINL float st_load1<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <> DL_DEVINL float st_load1<__half>(const __half* p) { return __half2float(*p); }
DL_DEVINL float st_max4(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }

DL_DEVINL void st_cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }      // cluster_wait() ends what it begins

// The row's work: what all CTAs of its cluster do together, or (local) one alone.
template <typename T, int THREADS> struct StRow {
    StShared& sh;
    const T* x;                        // the slice
    const int first, count;            // indexes first .. first + count - 1
    const bool wide;
    const int rank, ctas, tid, warp, lane;
    cg::cluster_group cluster;
    StScale scale;

    DL_DEVINL StShared* at(int r) const { return cluster.map_shared_rank(&sh, r); }

    // four logits from place i on (-inf behind the slice)
    DL_DEVINL float4 load(int i) const {
        if (i + 3 < count) return st_load4<T>(x + i, wide);
        float4 v = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
        if (i < count) v.x = st_load1<T>(x + i);
        if (i + 1 < count) v.y = st_load1<T>(x + i + 1);
        if (i + 2 < count) v.z = st_load1<T>(x + i + 2);
        return v;
    }
    // f(AH times four logits, the first one's place): the next four are `stride` behind it; whole warps, some loads in flight for each thread.  AH of one: a loop of one body
    template <int AH, typename F> DL_DEVINL void batches(int from, int to, int stride, F f) const {
        if constexpr (AH == 1) {
            float4 a{}, b{}, c{};
#pragma unroll 1
            for (int i = from - 3 * stride; i < to; i += stride) {
                const float4 v[1] = {a};
                a = b;
                b = c;
                c = load(i + 3 * stride + lane * 4);
                if (i >= from) f(v, i + lane * 4);
            }
        } else {
            for (int i = from; i < to; i += AH * stride) {
                float4 v[AH];
#pragma unroll
                for (int u = 0; u < AH; u++) v[u] = load(i + u * stride + lane * 4);
                f(v, i + lane * 4);
            }
        }
    }
    // f(four logits, the first one's place)
    template <int AH, typename F> DL_DEVINL void quads(int from, int to, int stride, F f) const {
        batches<AH>(from, to, stride, [&](const float4 (&v)[AH], int i) {
#pragma unroll
            for (int u = 0; u < AH; u++) f(v[u], i + u * stride);
        });
    }
    template <int AH, typename F> DL_DEVINL void all(F f) const { quads<AH>(warp * 128, count, THREADS * 4, f); }
    // f(logit, place) for what is not below `cut`; four neighbours a thread, most of which are passed over at once
    template <typename F> DL_DEVINL void each(float cut, F f) const {
        all<ST_AHEAD>([&](const float4& v, int i) {
            if (!(st_max4(v) >= cut) && cut > -CUDART_INF_F) return;
            const float e4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = e4[e] == e4[e] ? e4[e] : -CUDART_INF_F;      // (a NaN)
                if (y >= cut && i + e < count) f(y, i + e);
            }
        });
    }
    DL_DEVINL void add(int b, u64 w) {
        const unsigned w0 = (unsigned)w & 0x7fffu, w1 = (unsigned)(w >> 15) & 0x7fffu, w2 = (unsigned)(w >> 30);
        atomicAdd(&sh.hist[0][b], 1u);
        if (w0) atomicAdd(&sh.hist[1][b], w0);
        if (w1) atomicAdd(&sh.hist[2][b], w1);
        if (w2) atomicAdd(&sh.hist[3][b], w2);
    }
    DL_DEVINL void sync(bool local) {
        if (local) __syncthreads();
        else cluster.sync();
    }

    // The bin in which the weights reach the target (bin 0 is ahead of the others), of the CTA's bins or of the cluster's: sh.bin, sh.above.weight, sh.inside.  The bins are left empty.
    DL_DEVINL void locate(bool local, u64 ahead, u64 target) {
        static_assert(ST_BINS / 32 <= THREADS / 32 && ST_BINS <= 1024, "a warp for 32 bins");
        const bool mine = warp < ST_BINS / 32;
        StSums s = {0, 0};
        sync(local);
        if (local) {
            if (mine) s = StSums{(u64)sh.hist[1][tid] + ((u64)sh.hist[2][tid] << 15) + ((u64)sh.hist[3][tid] << 30), sh.hist[0][tid]};
        } else {
            const int share = ST_BINS / ctas;
            for (int j = tid; j < share * 4; j += THREADS) {   // four lanes a bin, one of its numbers each (a warp's lanes are all in or all out)
                const int part = j & 3, b = rank * share + (j >> 2);
                u64 x = 0;
#pragma unroll 8
                for (int r = 0; r < ctas; r++) x += at(r)->hist[part][b];
                const u64 n = __shfl_sync(0xffffffffu, x, lane & ~3);
                u64 w = part ? x << (15 * (part - 1)) : 0;
                w += __shfl_xor_sync(0xffffffffu, w, 1);
                w += __shfl_xor_sync(0xffffffffu, w, 2);
                for (int r = part; r < ctas; r += 4) at(r)->merged[b] = StSums{w, n};
            }
            cluster.sync();
            if (mine) s = sh.merged[tid];
        }
        u64 incl = s.weight;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 w = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += w;
        }
        if (lane == 31) sh.warp_sum[warp] = incl;
        if (mine) sh.hist[0][tid] = sh.hist[1][tid] = sh.hist[2][tid] = sh.hist[3][tid] = 0;
        if (tid == 0) sh.few = 0;
        __syncthreads();
        if (mine) {
            for (int w = 0; w < warp; w++) ahead += sh.warp_sum[w];
            const u64 to = ahead + incl, from = to - s.weight;
            if (from < target && to >= target) {
                sh.bin = tid;
                sh.above.weight = from;
                sh.inside = s;
            }
        }
        sync(local);                                            // (the cluster: `few` is zero everywhere)
    }

    // The first token, in an order, with which the sum of the weights reaches the target: its place in the order in sh.found, the sum up to it in sh.upto.  each(f) calls
    // f(order, bin, weight()) for every token that counts: larger orders are ahead, and so are lower bins; no two tokens have the same order.
    template <typename Each> DL_DEVINL void select(bool local, Each each, u64 target) {
        each([&](u64, int b, auto w) { add(b, w()); });
        locate(local, 0, target);
        u64 above = sh.above.weight, inside = sh.inside.count;
        const int bin = sh.bin;
        u64 lo = 0, hi = ~0ull;                                 // the orders in the bin
        bool range = false;                                    // they are known; `bin` is not looked at any more
        for (int turn = 0; turn < 8 && inside > ST_FEW; turn++) {      // (52 bits, eight at a time)
            if (!range) {
                u64 least = ~0ull, most = 0;
                each([&](u64 k, int b, auto) {
                    if (b != bin) return;
                    least = k < least ? k : least;
                    most = k > most ? k : most;
                });
                most = st_max_u64(most);
                least = ~st_max_u64(~least);
                if (lane == 0) { sh.red[warp].weight = most; sh.red[warp].count = least; }
                __syncthreads();
                for (int w = 0; w < THREADS / 32; w++) {
                    most = sh.red[w].weight > most ? sh.red[w].weight : most;
                    least = sh.red[w].count < least ? sh.red[w].count : least;
                }
                lo = least;
                hi = most;
                if (!local) {
                    if (tid < ctas) { at(tid)->lo[rank] = least; at(tid)->hi[rank] = most; }
                    cluster.sync();
                    for (int r = 0; r < ctas; r++) {
                        lo = sh.lo[r] < lo ? sh.lo[r] : lo;
                        hi = sh.hi[r] > hi ? sh.hi[r] : hi;
                    }
                }
                range = true;
            }
            const int bits = 64 - __clzll(hi - lo), shift = bits > 8 ? bits - 8 : 0;      // (hi > lo: more than one token)
            const u64 top = hi, end = lo;
            each([&](u64 k, int, auto w) { if (k <= top && k >= end) add((int)((top - k) >> shift), w()); });
            locate(local, above, target);
            above = sh.above.weight;
            inside = sh.inside.count;
            hi = top - ((u64)sh.bin << shift);
            const u64 width = (1ull << shift) - 1;
            lo = hi - end >= width ? hi - width : end;
        }
        each([&](u64 k, int b, auto w) {
            if (!(range ? k <= hi && k >= lo : b == bin)) return;
            const u64 wk = w();
            for (int r = local ? rank : 0; r < (local ? rank + 1 : ctas); r++) {      // (few tokens)
                StShared* o = at(r);
                const unsigned n = atomicAdd(&o->few, 1u);
                if (n < ST_FEW) { o->few_order[n] = k; o->few_weight[n] = wk; }
            }
        });
        sync(local);
        const int n = (int)min(inside, (u64)ST_FEW);
        for (int i = tid; i < n; i += THREADS) {
            const u64 k = sh.few_order[i];
            u64 s = above;
#pragma unroll 4
            for (int j = 0; j < n; j++)
                if (sh.few_order[j] > k) s += sh.few_weight[j];
            if (s < target && s + sh.few_weight[i] >= target) { sh.found = k; sh.upto = s + sh.few_weight[i]; }
        }
        __syncthreads();
    }

    // Tokens of AH quads go into this CTA's list (by whole warps): bit 4 u + e of `mask` is token e of the quad at place i + u * stride
    template <int AH> DL_DEVINL void push(unsigned mask, const float4 (&v)[AH], int i, int stride) {
        static_assert(AH <= 8, "a bit for each token");
        if (!__any_sync(0xffffffffu, mask)) return;
        const unsigned n = __popc(mask);
        unsigned incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        unsigned base = 0;
        if (lane == 31) base = atomicAdd(&sh.listed, incl);
        base = __shfl_sync(0xffffffffu, base, 31) + incl - n;
        if (!mask) return;
#pragma unroll
        for (int u = 0; u < AH; u++) {
            if (!(mask >> (4 * u) & 15)) continue;
            const float x4[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (mask >> (4 * u + e) & 1) {
                    if (base < ST_LIST) sh.list[base] = st_key(x4[e], first + i + u * stride + e);
                    base++;
                }
        }
    }
    // the CTAs' lists into CTA 0's
    DL_DEVINL void collect() {
        __syncthreads();
        if (rank != 0) {
            StShared* o = at(0);
            const unsigned n = min(sh.listed, (unsigned)ST_LIST);
            if (tid == 0) sh.few = atomicAdd(&o->others, sh.listed);
            __syncthreads();
            const unsigned from = sh.few;
            for (unsigned i = tid; i < n; i += THREADS)
                if (from + i < ST_LIST) o->list[ST_LIST - 1 - from - i] = sh.list[i];
        }
    }
    DL_DEVINL u64 listed(int i) const { return sh.list[i < (int)sh.listed ? i : ST_LIST - 1 - (i - (int)sh.listed)]; }
    // in which of n sums the target lies (sh.bin) and what the ones ahead of it add up to (sh.above.weight); n at most THREADS
    DL_DEVINL void locate_run(const u64* sums, int n, u64 target) {
        const u64 s = tid < n ? sums[tid] : 0;
        u64 incl = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; w++) incl += sh.warp_sum[w];
        if (incl - s < target && incl >= target) { sh.bin = tid; sh.above.weight = incl - s; }
        __syncthreads();
    }

    DL_DEVINL u64 sum(u64 v) {                                  // over the CTA, to all of its threads
        v = st_sum_u64(v);
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = v;
        __syncthreads();
        v = lane < THREADS / 32 ? sh.warp_sum[lane] : 0;
        return st_sum_u64(v);
    }
};

// What a row asks for.
struct StAsk {
    float m, T, p, min_p, coin, per;
    int k;
    bool by_k, by_p, by_min;
    double least;                      // min-p: logits that are not this far from the maximum stay

    // bins of the distance to the maximum: more than ST_REACH below it is the last one (whatever T: the distance is taken in units of it)
    DL_DEVINL int fine(float v) const { return v == m ? 0 : (int)fminf((m - v) * per, (float)(ST_FINE - 1)); }
    DL_DEVINL int bin(float v) const { return fine(v) / (ST_FINE / ST_BINS); }
    DL_DEVINL bool min_ok(float v) const { return !by_min || v == m || (double)v - (double)m >= least; }
    // the target of top-p
    DL_DEVINL u64 part(u64 total) const {
        bool more;
        const u64 t = st_times(total, p, more);
        return max(t + (more ? 1 : 0), 1ull);
    }
    // the coin's place: the token is the first one with which the sum is above it
    DL_DEVINL u64 want(u64 total) const {
        bool more;
        const u64 w = coin >= 1.f ? total - 1 : coin > 0.f ? st_times(total, coin, more) : 0;
        return w < total ? w : total - 1;
    }
    DL_DEVINL float prob(float v, u64 total) const { return (float)(exp(v == m ? 0. : ((double)v - (double)m) / (double)T) * 17592186044416.0 / (double)total); }
};

template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) sample_tokens_kernel(const __grid_constant__ StArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), row = blockIdx.x / ctas;
    StShared& sh = *reinterpret_cast<StShared*>(smem);
    const int first = rank * a.slice;
    StRow<T, THREADS> z{sh, reinterpret_cast<const T*>(a.logits) + (long long)row * a.ld + first, first, max(0, min(a.vocab - first, a.slice)), a.wide != 0,
                        rank, ctas, tid, tid >> 5, tid & 31, cluster, {0.f, 0.f, 0.f}};
    cluster_arrive_relaxed();                                   // (a CTA's shared memory is there once it has started: cluster_wait() ahead of the first store into another one's)
    pdl_launch_dependents();
    if (tid < 64) {
        const double p = exp2((double)tid / 64.0);
        sh.pow2[tid] = make_uint2((unsigned)__double2uint_rn(p * 2147483648.0), __float_as_uint((float)p));
    }
    if (tid == 64) { sh.listed = 0; sh.others = 0; sh.few = 0; sh.first = 0xffffffffu; }
    for (int b = tid; b < 4 * ST_BINS; b += THREADS) (&sh.hist[0][0])[b] = 0;
    pdl_wait();
    StAsk q;
    q.T = a.temperature[row];
    q.k = a.top_k ? a.top_k[row] : 0;
    q.p = a.top_p ? a.top_p[row] : 0.f;
    q.min_p = a.min_p ? a.min_p[row] : 0.f;
    q.coin = a.coin[row];
    // ---- the maximum ----
    float top = -CUDART_INF_F;
    z.template all<ST_AHEAD>([&](const float4& v, int) { top = fmaxf(top, st_max4(v)); });      // (no NaN)
    {
        float t = top;
#pragma unroll
        for (int g = 0; g < ST_LEVELS - 1; g++) {
            float l = t;
#pragma unroll
            for (int o = 1 << g; o < 32; o <<= 1) l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
            if (z.lane == 0) sh.warp_low[g][z.warp] = l;
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1 << g));
        }
        if (z.lane == 0) sh.warp_top[z.warp] = t;
    }
    __syncthreads();
    cluster_wait();
    if (tid < ctas * 8 && (tid & 7) < ST_LEVELS) {
        const int g = tid & 7, r = tid >> 3;
        const float* from = g < ST_LEVELS - 1 ? sh.warp_low[g] : sh.warp_top;
        float t = sh.warp_top[0], l = from[0];
        for (int w = 1; w < THREADS / 32; w++) {
            t = fmaxf(t, sh.warp_top[w]);
            l = fminf(l, from[w]);
        }
        StShared* o = z.at(r);
        o->low[g][rank] = l;
        if (g == 0) o->top[rank] = t;
    }
    cluster.sync();
    float m = sh.top[0];
    for (int r = 1; r < ctas; r++) m = fmaxf(m, sh.top[r]);
    q.m = m;
    if (!(q.T > 0.f) || m == -CUDART_INF_F) {                   // (uniform for the cluster) the first of the largest; token 0 where there is none
        if (m != -CUDART_INF_F) z.each(m, [&](float, int i) { atomicMin(&z.at(0)->first, (unsigned)(first + i)); });
        cluster.sync();
        if (rank == 0 && tid == 0) {
            a.tokens[row] = m == -CUDART_INF_F ? 0 : (int)sh.first;
            if (a.prob != nullptr) a.prob[row] = m == -CUDART_INF_F ? 0.f : 1.f;
        }
        return;
    }
    const double c = 1.4426950408889634 / (double)q.T;
    z.scale.m = m;
    z.scale.c_hi = (float)fmin(c, 3e38);
    z.scale.c_lo = c < 3e38 ? (float)(c - (double)z.scale.c_hi) : 0.f;
    q.per = z.scale.c_hi * (0.69314718f * (ST_FINE - 1) / ST_REACH);
    q.by_k = q.k > 0 && q.k < a.vocab;
    q.by_p = q.p > 0.f && q.p < 1.f;
    q.by_min = q.min_p > 0.f;
    q.least = q.by_min ? (double)q.T * log((double)fminf(q.min_p, 1.f)) : 0.;
    const float lowest = q.by_min ? fminf(m, __double2float_rd((double)m + q.least)) : -CUDART_INF_F;      // what is below, min-p takes out
    u64 border = 0;                                             // smallest key that stays
    constexpr int WARPS = THREADS / 32, AH = THREADS == 512 ? 1 : ST_AHEAD;      // quads a turn of top-p's passes (a row on sixteen CTAs: a turn or two, for which a long body is mostly code to be read: 23.7 and 22.0 us)
    const int run = ((a.slice + WARPS - 1) / WARPS + 127) / 128 * 128, r0 = z.warp * run, r1 = min(z.count, r0 + run);      // a warp's run of the slice

    // the weights of four neighbours that stay: not below the border, nor min-p's
    auto weights = [&](float cut, const float4& v4, int i, int end, u64 (&w)[4]) {
        w[0] = w[1] = w[2] = w[3] = 0;
        if (!(st_max4(v4) >= cut)) return;
        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (v[e] >= cut && i + e < end && st_key(v[e], first + i + e) >= border && q.min_ok(v[e])) w[e] = st_weight(v[e], z.scale, sh.pow2);
    };
    // the token: by the first CTA, in the run (CTA r's warp w's) that z.locate_run found; each warp takes a part of it
    auto draw_from = [&](int r, int w, u64 target, u64 total) {
        const int begin = r * a.slice, r_count = min(a.vocab - begin, a.slice), from = w * run, to = min(r_count, from + run);
        StRow<T, THREADS> y{sh, reinterpret_cast<const T*>(a.logits) + (long long)row * a.ld + begin, begin, r_count, z.wide, 0, ctas, tid, z.warp, z.lane, cluster, z.scale};
        const int part = ((run + WARPS - 1) / WARPS + 127) / 128 * 128, p0 = min(to, from + z.warp * part), p1 = min(to, p0 + part);
        const float cut = fmaxf(border ? st_logit(border) : -CUDART_INF_F, lowest);
        auto stays = [&](float v, int i, int end) -> u64 {
            return v >= cut && i < end && st_key(v, begin + i) >= border && q.min_ok(v) ? st_weight(v, z.scale, sh.pow2) : 0;
        };
        u64 before = sh.above.weight, mine = 0;
        for (int i0 = p0; i0 < p1; i0 += 128) {
            const int i = i0 + z.lane * 4;
            const float4 v = y.load(i);
            mine += (stays(v.x, i, p1) + stays(v.y, i + 1, p1)) + (stays(v.z, i + 2, p1) + stays(v.w, i + 3, p1));
        }
        mine = st_sum_u64(mine);
        __syncthreads();
        if (z.lane == 0) sh.warp_sum[z.warp] = mine;
        __syncthreads();
        for (int u = 0; u < z.warp; u++) before += sh.warp_sum[u];
        if (!(before < target && before + mine >= target)) return;
        for (int i0 = p0; i0 < p1; i0 += 128) {
            const int i = i0 + z.lane * 4;
            const float4 v4 = y.load(i);
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
            u64 we[4], s = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) { we[e] = stays(v[e], i + e, p1); s += we[e]; }
            u64 incl = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
                if (z.lane >= o) incl += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + incl >= target);
            if (hit) {
                if (z.lane == __ffs(hit) - 1) {
                    u64 at = before + incl - s;
                    bool there = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        at += we[e];
                        if (!there && at >= target) {
                            there = true;
                            a.tokens[row] = begin + i + e;
                            if (a.prob != nullptr) a.prob[row] = q.prob(v[e], total);
                        }
                    }
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    };

    if (q.by_k) {
        // ---- top-k: the list has all that can stay ----
        int groups = ST_LEVELS - 1;                             // the largest groups of which there are k
        while (groups >= 0 && q.k > ctas * THREADS >> groups) groups--;
        float cut = -CUDART_INF_F;
        if (groups >= 0) {
            cut = sh.low[groups][0];
            for (int r = 1; r < ctas; r++) cut = fminf(cut, sh.low[groups][r]);
        }
        // (of rows with masked tokens, or of a k beyond the maxima: all that is not -inf, which has no weight, whatever k is)
        const bool every = !(cut > -CUDART_INF_F);
        const float least = every ? -3.402823466e38f : cut;
        z.template batches<ST_AHEAD>(z.warp * 128, z.count, THREADS * 4, [&](const float4 (&v)[ST_AHEAD], int i) {
            unsigned mask = 0;
#pragma unroll
            for (int u = 0; u < ST_AHEAD; u++) {
                const int b = 4 * u;
                mask |= (v[u].x >= least ? 1u << b : 0) | (v[u].y >= least ? 2u << b : 0) | (v[u].z >= least ? 4u << b : 0) | (v[u].w >= least ? 8u << b : 0);
            }
            z.push(mask, v, i, THREADS * 4);
        });
        z.collect();
        cluster.sync();
        if (rank == 0) {
            const unsigned found = sh.listed + sh.others;
            const int n = (int)min(found, (unsigned)ST_LIST);
            const bool ok = found <= ST_LIST && (every || n >= q.k);
            if (tid < ctas) z.at(tid)->done = ok ? 1 : 0;       // (the others may leave)
            st_cluster_arrive();
            if (ok) {
                const float per = !every ? (float)(ST_BINS - 1) / (m - cut) : q.per / (ST_FINE / ST_BINS);      // (bins from the maximum to the least of the list; infinities: some bin, the same for equal ones)
                auto by_logit = [&](bool counts) {              // the list in the order of the logits, from the border on
                    return [&, counts](auto f) {
                        for (int i = tid; i < n; i += THREADS) {
                            const u64 key = z.listed(i);
                            const float v = st_logit(key);
                            if (key >= border) f(key, v == m ? 0 : (int)fminf((m - v) * per, (float)(ST_BINS - 1)), [&] { return counts ? 1 : st_weight(v, z.scale, sh.pow2); });
                        }
                    };
                };
                auto left = [&](bool min_too) {                  // the weight of what stays
                    u64 s = 0;
                    for (int i = tid; i < n; i += THREADS) {
                        const u64 key = z.listed(i);
                        const float v = st_logit(key);
                        if (key >= border && (!min_too || q.min_ok(v))) s += st_weight(v, z.scale, sh.pow2);
                    }
                    return z.sum(s);
                };
                if (q.k < n) {
                    z.select(true, by_logit(true), (u64)q.k);
                    border = sh.found;
                }
                if (q.by_p) {
                    z.select(true, by_logit(false), q.part(left(false)));
                    border = sh.found;
                }
                const u64 kept = left(true);
                const int per_bin = (a.vocab + ST_BINS - 1) / ST_BINS;
                z.select(true, [&](auto f) {                     // in the order of the vocabulary
                    for (int i = tid; i < n; i += THREADS) {
                        const u64 key = z.listed(i);
                        const float v = st_logit(key);
                        if (key >= border && q.min_ok(v)) f(key & ST_IDX_MASK, st_index(key) / per_bin, [&] { return st_weight(v, z.scale, sh.pow2); });
                    }
                }, q.want(kept) + 1);
                if (a.prob != nullptr)
                    for (int i = tid; i < n; i += THREADS)
                        if ((z.listed(i) & ST_IDX_MASK) == sh.found) a.prob[row] = q.prob(st_logit(z.listed(i)), kept);
                if (tid == 0) a.tokens[row] = (int)(ST_IDX_MASK - sh.found);
            }
        } else {
            st_cluster_arrive();
        }
        cluster_wait();
        if (sh.done) return;
    } else {
        // ---- top-p: the bins in which the border has to lie; where there is none, no bin ----
        int from = ST_FINE, to = -1;
        if (q.by_p) {
            const float width = ST_REACH / (ST_FINE - 1);
            float more = 0.f;                                   // what the tokens of the heavy bins weigh beyond the middle of their bin, in widths of a bin
            for (int b = tid; b < ST_FINE; b += THREADS) sh.count.fine[b] = 0;
            __syncthreads();
            z.template all<AH>([&](const float4& v4, int i) {
                const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float t = (m - v[e]) * q.per;
                    if (t < (float)(ST_FINE - 1)) atomicAdd(&sh.count.fine[(int)t], 1u);      // (what is farther, or no number, has next to no weight)
                    if (t < (float)ST_HEAVY) more = fmaf(__expf(-width * t), 0.5f - (t - truncf(t)), more);
                }
            });
            more = warp_sum(more);
            if (z.lane == 0) sh.warp_low[1][z.warp] = more;
            cluster.sync();
            if (z.warp == WARPS - 1) {
                more = warp_sum(z.lane < WARPS ? sh.warp_low[1][z.lane] : 0.f);
                if (z.lane < ctas) z.at(z.lane)->low[0][rank] = more;
            }
            const int share = ST_FINE / ctas;
            for (int j = tid; j < share; j += THREADS) {
                unsigned s = 0;
#pragma unroll 8
                for (int r = 0; r < ctas; r++) s += z.at(r)->count.fine[rank * share + j];
                for (int r = 0; r < ctas; r++) z.at(r)->count.fine_sum[rank * share + j] = s;
            }
            if (tid == 0) { sh.bin_from = 0; sh.bin_to = ST_FINE - 1; }
            cluster.sync();
            // sums from the counts, each bin's tokens in its middle; off by a random part of the width for each bin (16-bit logits: a bin's tokens have one value).  A few heavy tokens would make most of
            // that: behind the heavy bins theirs are known
            constexpr int PER = (ST_FINE + THREADS - 1) / THREADS;
            float w[PER], part = 0.f, off = 0.f, off_light = 0.f;
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const int b = tid * PER + e;
                const float n = b < ST_FINE ? (float)sh.count.fine_sum[b] : 0.f, mid = __expf(-((float)b + 0.5f) * width);
                w[e] = n * mid;
                part += w[e];
                off += w[e] * w[e];
                off_light += b >= ST_HEAVY ? w[e] * w[e] : 0.f;
            }
            float incl = part;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float y = __shfl_up_sync(0xffffffffu, incl, o);
                if (z.lane >= o) incl += y;
            }
            off = warp_sum(off);
            off_light = warp_sum(off_light);
            if (z.lane == 31) { sh.warp_top[z.warp] = incl; sh.warp_low[0][z.warp] = off; sh.warp_low[2][z.warp] = off_light; }
            __syncthreads();
            float ahead = incl - part, all = 0.f;
            off = off_light = more = 0.f;
            for (int u = 0; u < WARPS; u++) {
                if (u < z.warp) ahead += sh.warp_top[u];
                all += sh.warp_top[u];
                off += sh.warp_low[0][u];
                off_light += sh.warp_low[2][u];
            }
            for (int r = 0; r < ctas; r++) more += sh.low[0][r];
            more *= width;
            all += more;
            // four standard deviations (width / sqrt 12 of a bin's weight), e^-20 for each token of the tail, and the sums' roundings
            const float tail = 2.1e-9f * (float)a.vocab + all * 0x1p-17f, room = 1.2f * width * sqrtf(off) + tail, room_light = 1.2f * width * sqrtf(off_light) + tail, goal = q.p * all;
            // the last bin that begins ahead of the target for sure, the first one that ends behind it
            int f_b = 0, t_b = ST_FINE - 1;
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const int b = tid * PER + e;
                if (b < ST_FINE) {
                    if (b < ST_HEAVY ? ahead + room < goal : ahead + more + room_light < goal) f_b = b;
                    const float end = ahead + w[e];
                    if (b < t_b && (b + 1 < ST_HEAVY ? end - room >= goal : end + more - room_light >= goal)) t_b = b;
                }
                ahead += w[e];
            }
            f_b = __reduce_max_sync(0xffffffffu, f_b);
            t_b = __reduce_min_sync(0xffffffffu, t_b);
            if (z.lane == 0) { atomicMax(&sh.bin_from, f_b); atomicMin(&sh.bin_to, t_b); }
            __syncthreads();
            from = sh.bin_from;
            to = max(from, sh.bin_to);
            cluster.sync();                                     // (the list takes the counts' place)
        }
        // ---- the weights: of all that is ahead of those bins, by runs, and of the row ----
        // (a run ends with a whole quad or with the slice, behind which logits are -inf)
        u64 mine = 0, ahead = 0, all = 0;                        // what is drawn from, what is ahead of the border's bins, the row
        const float from_t = (float)from, to_t = to == ST_FINE - 1 ? CUDART_INF_F : (float)(to + 1);
        z.template batches<AH>(r0, r1, 128, [&](const float4 (&v4)[AH], int i) {
            unsigned mask = 0;
#pragma unroll
            for (int u = 0; u < AH; u++) {
                const float v[4] = {v4[u].x, v4[u].y, v4[u].z, v4[u].w};
                if (i - z.lane * 4 + u * 128 >= r1) break;       // (uniform for the warp)
                if (to < 0) {
                    if (!(st_max4(v4[u]) >= lowest)) continue;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!q.by_min || (v[e] >= lowest && q.min_ok(v[e]))) mine += st_weight(v[e], z.scale, sh.pow2);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u64 w = st_weight_below(v[e], z.scale, sh.pow2);      // (of the maximum, too: it is finite)
                    const float t = (m - v[e]) * q.per;          // (fine())
                    const bool front = t < from_t;
                    all += w;
                    ahead += front ? w : 0;
                    if (q.by_min) mine += front && v[e] >= lowest && q.min_ok(v[e]) ? w : 0;
                    mask |= t >= from_t && t < to_t ? 1u << (4 * u + e) : 0;
                }
            }
            if (to >= 0) z.push(mask, v4, i, 128);
        });
        if (to >= 0 && !q.by_min) mine = ahead;
        if (to >= 0) z.collect();
        mine = st_sum_u64(mine);
        if (z.lane == 0) z.at(0)->run_sum[rank * WARPS + z.warp] = mine;
        if (to >= 0) {
            ahead = z.sum(ahead);
            all = z.sum(all);
            if (tid == 0) { z.at(0)->cta_sum[rank] = ahead; z.at(0)->lo[rank] = all; }
        }
        cluster.sync();
        if (rank == 0) {
            bool ok = true;
            if (to >= 0) {
                const unsigned found = sh.listed + sh.others;
                const int n = (int)min(found, (unsigned)ST_LIST);
                u64 total = 0, near = 0;
                ahead = 0;
                for (int r = 0; r < ctas; r++) { ahead += sh.cta_sum[r]; total += sh.lo[r]; }
                for (int i = tid; i < n; i += THREADS) near += st_weight(st_logit(z.listed(i)), z.scale, sh.pow2);
                near = z.sum(near);
                const u64 target = q.part(total);
                ok = m < CUDART_INF_F && found <= ST_LIST && ahead < target && target <= ahead + near;
                if (ok) {
                    const int wide = (to - from) / ST_BINS + 1;      // fine bins to one of select's
                    z.select(true, [&](auto f) {
                        for (int i = tid; i < n; i += THREADS) {
                            const u64 key = z.listed(i);
                            const float v = st_logit(key);
                            f(key, (q.fine(v) - from) / wide, [&] { return st_weight(v, z.scale, sh.pow2); });
                        }
                    }, target - ahead);
                    border = sh.found;
                    for (int i = tid; i < n; i += THREADS) {         // those of the list that stay, to their runs
                        const u64 key = z.listed(i);
                        const float v = st_logit(key);
                        const int at = st_index(key), r = at / a.slice;
                        if (key >= border && q.min_ok(v)) atomicAdd(&sh.run_sum[r * WARPS + (at - r * a.slice) / run], st_weight(v, z.scale, sh.pow2));
                    }
                    __syncthreads();
                }
            }
            if (tid < ctas && to >= 0) z.at(tid)->done = ok ? 1 : 0;      // (the others may leave)
            st_cluster_arrive();
            if (ok) {
                const int n = ctas * WARPS;
                const u64 kept = z.sum(tid < n ? sh.run_sum[tid] : 0), target = q.want(kept) + 1;
                z.locate_run(sh.run_sum, n, target);
                draw_from(sh.bin / WARPS, sh.bin % WARPS, target, kept);
            }
        } else {
            st_cluster_arrive();
        }
        cluster_wait();
        if (to < 0 || sh.done) return;
    }
    // ---- the same over the whole row, by all CTAs ----
    border = 0;
    auto by_logit = [&](bool counts) {
        return [&, counts](auto f) {
            z.each(border ? st_logit(border) : -CUDART_INF_F, [&](float v, int i) {
                const u64 key = st_key(v, first + i);
                if (key >= border) f(key, q.bin(v), [&] { return counts ? 1 : st_weight(v, z.scale, sh.pow2); });
            });
        };
    };
    if (q.by_k) {
        z.select(false, by_logit(true), (u64)q.k);
        border = sh.found;
    }
    if (q.by_p) {
        u64 left = 0, total = 0;
        z.each(border ? st_logit(border) : -CUDART_INF_F, [&](float v, int i) { if (st_key(v, first + i) >= border) left += st_weight(v, z.scale, sh.pow2); });
        left = z.sum(left);
        if (tid < ctas) z.at(tid)->cta_sum[rank] = left;
        cluster.sync();
        for (int r = 0; r < ctas; r++) total += sh.cta_sum[r];
        z.select(false, by_logit(false), q.part(total));
        border = sh.found;
    }
    u64 mine = 0;
    z.template quads<ST_AHEAD>(r0, r1, 128, [&](const float4& v, int i) {
        u64 w[4];
        weights(fmaxf(border ? st_logit(border) : -CUDART_INF_F, lowest), v, i, r1, w);
        mine += (w[0] + w[1]) + (w[2] + w[3]);
    });
    mine = st_sum_u64(mine);
    if (z.lane == 0) z.at(0)->run_sum[rank * WARPS + z.warp] = mine;
    cluster.sync();
    if (rank != 0) return;
    const int n = ctas * WARPS;
    const u64 kept = z.sum(tid < n ? sh.run_sum[tid] : 0), target = q.want(kept) + 1;
    z.locate_run(sh.run_sum, n, target);
    draw_from(sh.bin / WARPS, sh.bin % WARPS, target, kept);
}

extern void dl_set_error(const char* fmt, ...);
extern "C" int dl_device_sm_count();

template <typename T, int THREADS, int PER_SM> static int st_launch(const StArgs& a, int M, int ctas, int pdl, cudaStream_t stream) {
    static SmemLimit given;
    auto* kernel = sample_tokens_kernel<T, THREADS, PER_SM>;
    if (const int rc = dl_smem_limit("dl_sample_tokens", kernel, sizeof(StShared), given)) return rc;
    static SmemLimit wide_clusters;                             // (clusters of more than eight: a setting of each device, too)
    if (ctas > 8) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess && (dev >= 64 || wide_clusters.bytes[dev] == 0)) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) { dl_set_error("dl_sample_tokens cluster attr: %s", cudaGetErrorString(e)); return -(int)e; }
        if (dev < 64) wide_clusters.bytes[dev] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(M * ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sizeof(StShared);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) { dl_set_error("dl_sample_tokens launch: %s", cudaGetErrorString(e)); return -(int)e; }
    return 0;
}

// Largest vocabulary of dl_sample_tokens: its weights' sum fits 64 bits
extern "C" int dl_sample_tokens_max_vocab() { return 1 << 19; }

extern "C" int dl_sample_tokens(const void* logits, int type, int M, int vocab, long long ld, const float* temperature, const int* top_k, const float* top_p, const float* min_p, const float* coin,
                                int* tokens_out, float* prob_out, int pdl, void* stream) {
    if (M < 0 || vocab < 1 || vocab > dl_sample_tokens_max_vocab() || M > 1 << 24) { dl_set_error("dl_sample_tokens: %d rows of %d logits (at most %d)", M, vocab, dl_sample_tokens_max_vocab()); return -1; }
    if (ld < vocab && M > 1) { dl_set_error("dl_sample_tokens: rows overlap (ld %lld)", ld); return -1; }
    if (type != 0 && type != 1 && type != 2) { dl_set_error("dl_sample_tokens: unsupported type %d", type); return -1; }
    if (M == 0) return 0;
    if (!logits || !temperature || !coin || !tokens_out) { dl_set_error("dl_sample_tokens: a null pointer"); return -1; }
    // CTAs of a row: what leaves the fullest SM least to do, the fewer the better; 4096 logits a CTA or more, 131072 at most (a bin's parts of 15 bits fit 32)
    const int n_sms = dl_device_sm_count() > 0 ? dl_device_sm_count() : 1;
    int ctas = 1;
    double least = 1e30;
    for (int c = 1; c <= ST_MAX_CTAS && (c == 1 || vocab >= c * 4096); c *= 2) {
        if (c > 8 && (long long)M * c > n_sms / 2) break;      // (sixteen of them want most of a GPC)
        if (vocab > c * 131072) continue;
        const double load = (double)(((long long)M * c + n_sms - 1) / n_sms) / c;
        if (load < 0.85 * least) { least = load; ctas = c; }
    }
    const int slice = ((vocab + ctas - 1) / ctas + 31) / 32 * 32;
    const int group = type == 0 ? 16 : 8;
    const bool wide = ((uintptr_t)logits % group) == 0 && (M == 1 || ld * (group / 4) % group == 0);
    const StArgs a = {logits, ld, temperature, top_p, min_p, coin, top_k, tokens_out, prob_out, vocab, slice, wide ? 1 : 0};
    cudaStream_t st = (cudaStream_t)stream;
    // few rows: an SM for each CTA, and all of its threads; half of them where the cluster is so large that its barriers cost more (one row, top-p: 22.2 us with 512, 24.9 with 1024; eight rows,
    // top-k and top-p, in clusters of eight: 23.7 and 19.6)
    const int variant = (long long)M * ctas > n_sms ? 0 : ctas > 8 ? 1 : 2;
    auto go = [&](auto zero) {
        using T = decltype(zero);
        return variant == 0 ? st_launch<T, 384, 3>(a, M, ctas, pdl, st) : variant == 1 ? st_launch<T, 512, 1>(a, M, ctas, pdl, st) : st_launch<T, 1024, 1>(a, M, ctas, pdl, st);
    };
    if (type == 0) return go(float());
    if (type == 1) return go(__nv_bfloat16());
    return go(__half());
}
