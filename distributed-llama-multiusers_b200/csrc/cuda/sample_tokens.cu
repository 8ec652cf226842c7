// A token for every row of logits from given random numbers: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T); the order of tokens: largest logit first, of equal ones the lowest index first
//   top-k   a token stays if fewer than k are ahead of it;
//   top-p   of those a token stays if the weight ahead of it is below p times the weight of what top-k leaves;
//   min-p   of those a token stays if w_i >= min_p (the largest weight is 1)
//   the token: in the order of the vocabulary the first one where the sum of the weights that stay is above coin times their total
// so what stays is always the front of the order, and one border (logit, index) tells it.  T <= 0: the first of the largest.
//
// A cluster of CTAs per row holds the row's logits in shared memory, read from memory once.  The border is found without sorting: 256 bins of the distance
// to the maximum with their counts and weights, summed over the cluster, give the bin in which the border lies, and its few tokens are compared with each other.  Where a bin
// holds more than the list takes (logits that are equal, or far below the maximum) it is divided again, by the bits of logit and index together, which
// no two tokens share, until it fits.
//
// Weights are whole numbers of 2^-44, so that sums do not depend on their order; they are exact to 2^-29 of themselves (a table of 64 powers of two and a
// polynomial, after P. T. P. Tang's table-driven exponential, on the difference and the factor as pairs of f32 numbers): with sums of f32 results a
// coin next to a border between two tokens would fall on the other side once in some thousand rows.
#include <math_constants.h>
#include <cuda_bf16.h>
#include "common.cuh"
#include "smem_limit.cuh"

#define ST_BINS 256
#define ST_LIST 512
#define ST_MAX_CTAS 8
#define ST_REACH 10.0f                 // the bins' range below the maximum, in units of the exponent
#define ST_IDX_BITS 20
#define ST_ONE (1ull << 44)
#define ST_MAX_SLICE 40960             // logits of a CTA

typedef unsigned long long u64;

struct StArgs {
    const void* logits;
    long long ld;
    const float *temperature, *top_p, *min_p, *coin;
    const int* top_k;
    int* tokens;
    float* prob;
    int vocab, slice;
    int wide;                          // rows can be read 16 bytes at a time
};

struct StSums { u64 weight; u64 count; };

// what the CTAs of a row leave for each other; in each CTA's shared memory, ahead of its slice
struct alignas(16) StShared {
    union {
        unsigned hist[4][ST_BINS];     // this CTA's counts, and weights in three parts of 15 bits
        u64 list_key[ST_LIST];         // later: the tokens of the border's bin, the cluster's
    };
    union {
        StSums merged[ST_BINS];        // the cluster's bins
        u64 list_weight[ST_LIST];
    };
    u64 key[ST_MAX_CTAS];              // each CTA's largest
    u64 lo[ST_MAX_CTAS], hi[ST_MAX_CTAS];
    u64 cta_sum[ST_MAX_CTAS];
    StSums above, inside;              // of the bin found: what lies ahead of it and in it
    int bin;
    unsigned listed;
    u64 border;                        // smallest key that stays
    u64 warp_sum[32];
    StSums red[32];
    uint2 pow2[64];                    // 2^(j / 64): times 2^31, and as f32
};
static_assert(sizeof(StShared) + ST_MAX_SLICE * 4 <= 227 * 1024, "a slice and what goes with it fit an SM");

DL_DEVINL unsigned st_order(float x) {
    const unsigned b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
// logit and index as one number, larger for what is ahead
DL_DEVINL u64 st_key(float x, int i) { return ((u64)st_order(x) << ST_IDX_BITS) | (u64)((1 << ST_IDX_BITS) - 1 - i); }

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
    const float d = x - s.m, p = d * s.c_hi;
    const float b = d - x, lost = (x - (d - b)) + (-s.m - b);   // x - m = d + lost
    const float e = fmaf(lost, s.c_hi, fmaf(d, s.c_lo, fmaf(d, s.c_hi, -p)));
    const float t = p + 196608.f;                              // 1.5 2^17: p to the nearest 1 / 64
    const int k = __float_as_int(t) - __float_as_int(196608.f);
    const float r = (p - (t - 196608.f)) + e;                   // at most 2^-7
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

// The row's work: what all CTAs of its cluster do together.
template <int THREADS> struct StRow {
    StShared& sh;
    const float* x;
    const int first, count;            // the slice: indexes first .. first + count - 1
    const int rank, ctas, tid, warp, lane;
    cg::cluster_group cluster;
    StScale scale;

    DL_DEVINL StShared* at(int r) const { return cluster.map_shared_rank(&sh, r); }

    // f(logit, place in the slice) for what is not below `cut` (and may be for others); four neighbours a thread, most of which are passed over at once
    template <typename F> DL_DEVINL void each(float cut, F f) const {
        for (int i = tid * 4; i < count; i += THREADS * 4) {
            const float4 v = *reinterpret_cast<const float4*>(x + i);
            if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= cut)) continue;      // (behind the slice: anything)
            const float e4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e4[e] >= cut && i + e < count) f(e4[e], i + e);
        }
    }
    DL_DEVINL void clear() {
        for (int b = tid; b < 4 * ST_BINS; b += THREADS) (&sh.hist[0][0])[b] = 0;
    }
    DL_DEVINL void add(int b, unsigned n, u64 w, bool weights) {
        atomicAdd(&sh.hist[0][b], n);
        if (weights) {
            const unsigned w0 = (unsigned)w & 0x7fffu, w1 = (unsigned)(w >> 15) & 0x7fffu, w2 = (unsigned)(w >> 30);
            if (w0) atomicAdd(&sh.hist[1][b], w0);
            if (w1) atomicAdd(&sh.hist[2][b], w1);
            if (w2) atomicAdd(&sh.hist[3][b], w2);
        }
    }

    // The CTAs' bins added up, in every CTA's sh.merged.
    DL_DEVINL void merge() {
        cluster.sync();
        const int share = ST_BINS / ctas;
        for (int j = tid; j < share * 4; j += THREADS) {       // four lanes a bin, one of its numbers each (a warp's lanes are all in or all out)
            const int part = j & 3, b = rank * share + (j >> 2);
            u64 s = 0;
#pragma unroll
            for (int r = 0; r < ST_MAX_CTAS; r++)
                if (r < ctas) s += at(r)->hist[part][b];
            const u64 n = __shfl_sync(0xffffffffu, s, lane & ~3);
            u64 w = part ? s << (15 * (part - 1)) : 0;
            w += __shfl_xor_sync(0xffffffffu, w, 1);
            w += __shfl_xor_sync(0xffffffffu, w, 2);
            for (int r = part; r < ctas; r += 4) at(r)->merged[b] = StSums{w, n};
        }
        if (tid == 0) sh.listed = 0;
        cluster.sync();
    }

    // The bin in which what lies ahead reaches the target (bin 0 is ahead of the others): sh.bin, sh.above, sh.inside; each CTA for itself.
    DL_DEVINL void locate(const StSums& ahead, bool by_weight, u64 target) {
        static_assert(ST_BINS / 32 <= THREADS / 32 && ST_BINS <= 1024, "a warp for 32 bins");
        const bool mine = warp < ST_BINS / 32;
        StSums s = {0, 0}, incl;
        if (mine) s = sh.merged[warp * 32 + lane];
        incl = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 c = __shfl_up_sync(0xffffffffu, incl.count, o), w = __shfl_up_sync(0xffffffffu, incl.weight, o);
            if (lane >= o) { incl.count += c; incl.weight += w; }
        }
        if (lane == 31) sh.red[warp] = incl;
        __syncthreads();
        if (mine) {
            StSums before = ahead;
            for (int w = 0; w < warp; w++) { before.count += sh.red[w].count; before.weight += sh.red[w].weight; }
            const u64 to = by_weight ? before.weight + incl.weight : before.count + incl.count, from = to - (by_weight ? s.weight : s.count);
            if (from < target && to >= target) {
                sh.bin = warp * 32 + lane;
                sh.above = StSums{before.weight + incl.weight - s.weight, before.count + incl.count - s.count};
                sh.inside = s;
            }
        }
        __syncthreads();
    }

    // The border for a target: the key of the first token with which the sums reach it, in every CTA's sh.border.  `bin_of` gave the bins in place, cut_of(bin) is a logit that what is in
    // the bin is not below.
    template <typename Bin, typename Cut> DL_DEVINL void select(Bin bin_of, Cut cut_of, bool by_weight, u64 target) {
        locate(StSums{0, 0}, by_weight, target);
        StSums above = sh.above, inside = sh.inside;
        const int bin = sh.bin;
        const float cut = cut_of(bin);
        u64 lo = 0, hi = ~0ull;                                 // the keys of the bin
        bool range = false;                                    // they are known; `bin` is not looked at any more
        for (int turn = 0; turn < 8 && inside.count > ST_LIST; turn++) {      // (52 bits of key, eight at a time)
            if (!range) {
                u64 least = ~0ull, most = 0;
                each(cut, [&](float v, int i) {
                    if (bin_of(v, first + i) == bin) {
                        const u64 k = st_key(v, first + i);
                        least = k < least ? k : least;
                        most = k > most ? k : most;
                    }
                });
                most = st_max_u64(most);
                least = ~st_max_u64(~least);
                if (lane == 0) { sh.red[warp].weight = most; sh.red[warp].count = least; }
                __syncthreads();
                if (tid < ctas) {
                    for (int w = 0; w < THREADS / 32; w++) {
                        most = sh.red[w].weight > most ? sh.red[w].weight : most;
                        least = sh.red[w].count < least ? sh.red[w].count : least;
                    }
                    at(tid)->lo[rank] = least;
                    at(tid)->hi[rank] = most;
                }
                cluster.sync();
                lo = ~0ull; hi = 0;
                for (int r = 0; r < ctas; r++) {
                    lo = sh.lo[r] < lo ? sh.lo[r] : lo;
                    hi = sh.hi[r] > hi ? sh.hi[r] : hi;
                }
                range = true;
            }
            const int bits = 64 - __clzll(hi - lo), shift = bits > 8 ? bits - 8 : 0;      // (hi > lo: more than one token)
            const u64 top = hi, end = lo;
            clear();
            __syncthreads();
            each(cut, [&](float v, int i) {
                const u64 k = st_key(v, first + i);
                if (k <= top && k >= end) add((int)((top - k) >> shift), 1, by_weight ? st_weight(v, scale, sh.pow2) : 0, by_weight);
            });
            merge();
            locate(above, by_weight, target);
            above = sh.above;
            inside = sh.inside;
            hi = top - ((u64)sh.bin << shift);
            const u64 width = (1ull << shift) - 1;
            lo = hi - end >= width ? hi - width : end;
        }
        each(cut, [&](float v, int i) {
            const u64 k = st_key(v, first + i);
            if (!(range ? k <= hi && k >= lo : bin_of(v, first + i) == bin)) return;
            for (int r = 0; r < ctas; r++) {                   // (few tokens)
                StShared* o = at(r);
                const unsigned n = atomicAdd(&o->listed, 1u);
                if (n < ST_LIST) o->list_key[n] = k;
            }
        });
        cluster.sync();
        const int n = (int)min(inside.count, (u64)ST_LIST);
        if (by_weight)
            for (int i = tid; i < n; i += THREADS) {
                const unsigned q = (unsigned)(sh.list_key[i] >> ST_IDX_BITS);
                sh.list_weight[i] = st_weight(__uint_as_float((q & 0x80000000u) ? q ^ 0x80000000u : ~q), scale, sh.pow2);
            }
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
            const u64 k = sh.list_key[i];
            u64 s = by_weight ? above.weight : above.count;
#pragma unroll 4
            for (int j = 0; j < n; j++)
                if (sh.list_key[j] > k) s += by_weight ? sh.list_weight[j] : 1;
            if (s < target && s + (by_weight ? sh.list_weight[i] : 1) >= target) sh.border = k;
        }
        __syncthreads();
    }
};

template <typename T> DL_DEVINL float st_value(T v);
template <> DL_DEVINL float st_value<float>(float v) { return v; }
template <> DL_DEVINL float st_value<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> DL_DEVINL float st_value<__half>(__half v) { return __half2float(v); }

template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) sample_tokens_kernel(const __grid_constant__ StArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), row = blockIdx.x / ctas;
    StShared& sh = *reinterpret_cast<StShared*>(smem);
    float* x = reinterpret_cast<float*>(smem + sizeof(StShared));
    const int first = rank * a.slice;
    StRow<THREADS> z{sh, x, first, max(0, min(a.vocab - first, a.slice)), rank, ctas, tid, tid >> 5, tid & 31, cluster, {0.f, 0.f, 0.f}};
    pdl_launch_dependents();
    if (tid < 64) {
        const double p = exp2((double)tid / 64.0);
        sh.pow2[tid] = make_uint2((unsigned)__double2uint_rn(p * 2147483648.0), __float_as_uint((float)p));
    }
    z.clear();
    pdl_wait();
    // ---- the slice into shared memory, and the first of the largest ----
    const T* src = reinterpret_cast<const T*>(a.logits) + (long long)row * a.ld + first;
    float top = -CUDART_INF_F;
    int top_i = 0x7fffffff;
    auto take = [&](float v, int i) {
        v = v == v ? v + 0.f : -CUDART_INF_F;                   // no NaN, no negative zero
        if (v > top || top_i == 0x7fffffff) { top = v; top_i = i; }      // (a thread's places ascend)
        return v;
    };
    if (a.wide) {
        constexpr int PER = 16 / sizeof(T);
        const int whole = z.count / PER * PER;
#pragma unroll 4
        for (int i = tid * PER; i < whole; i += THREADS * PER) {
            const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(src + i));
            float v[PER];
#pragma unroll
            for (int e = 0; e < PER; e++) v[e] = take(st_value<T>(reinterpret_cast<const T*>(&raw)[e]), i + e);
#pragma unroll
            for (int e = 0; e < PER; e += 4) *reinterpret_cast<float4*>(x + i + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
        if (whole + tid < z.count) x[whole + tid] = take(st_value<T>(src[whole + tid]), whole + tid);
    } else {
#pragma unroll 8
        for (int i = tid; i < z.count; i += THREADS) x[i] = take(st_value<T>(src[i]), i);
    }
    u64 best = top_i == 0x7fffffff ? 0 : st_key(top, first + top_i);
    best = st_max_u64(best);
    if (z.lane == 0) sh.warp_sum[z.warp] = best;
    __syncthreads();
    if (tid < ctas) {
        for (int w = 0; w < (THREADS / 32); w++) best = sh.warp_sum[w] > best ? sh.warp_sum[w] : best;
        cluster.map_shared_rank(&sh, tid)->key[rank] = best;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < ctas; r++) best = sh.key[r] > best ? sh.key[r] : best;
    const unsigned o = (unsigned)(best >> ST_IDX_BITS);
    const float m = __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
    const float T0 = a.temperature[row];
    if (!(T0 > 0.f) || m == -CUDART_INF_F) {                    // (uniform for the cluster; nobody reads another's memory any more)
        if (rank == 0 && tid == 0) {
            a.tokens[row] = (1 << ST_IDX_BITS) - 1 - (int)(best & ((1 << ST_IDX_BITS) - 1));
            if (a.prob != nullptr) a.prob[row] = m == -CUDART_INF_F ? 0.f : 1.f;
        }
        return;
    }
    const double c = 1.4426950408889634 / (double)T0;
    z.scale.m = m;
    z.scale.c_hi = (float)fmin(c, 3e38);
    z.scale.c_lo = c < 3e38 ? (float)(c - (double)z.scale.c_hi) : 0.f;

    // ---- the border of top-k and top-p ----
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 0.f;
    const float min_p = a.min_p ? a.min_p[row] : 0.f;
    const bool by_k = k > 0 && k < a.vocab, by_p = p > 0.f && p < 1.f;
    u64 border = 0;
    // bins of the distance to the maximum: more than ST_REACH below it is the last one (whatever T: the distance is taken in units of it)
    const float per = z.scale.c_hi * (0.69314718f * (ST_BINS - 1) / ST_REACH);
    auto bin_of = [=](float v, int) { return v == m ? 0 : (int)fminf((m - v) * per, (float)(ST_BINS - 1)); };
    auto cut_of = [=](int bin) {                                // (1e-5 of room for the roundings; a row of which nothing can be said: all of it)
        const float far = (float)(bin + 1) / per * 1.00001f, c = m - far - fabsf(m) * 1e-6f;
        return bin < ST_BINS - 1 && per > 0.f && c == c ? c : -CUDART_INF_F;
    };
    if (by_k) {
        unsigned n = 0;
        z.each(cut_of(ST_BINS - 2), [&](float v, int i) {
            const int b = bin_of(v, 0);
            if (b < ST_BINS - 1) { atomicAdd(&sh.hist[0][b], 1u); n++; }
        });
        n = __reduce_add_sync(0xffffffffu, n);
        if (z.lane == 0 && n) atomicAdd(&sh.hist[1][ST_BINS - 1], n);      // (counts alone: the other parts are free)
        __syncthreads();
        if (tid == 0) {
            sh.hist[0][ST_BINS - 1] = (unsigned)z.count - sh.hist[1][ST_BINS - 1];      // the rest
            sh.hist[1][ST_BINS - 1] = 0;
        }
        z.merge();
        z.select(bin_of, cut_of, false, (u64)k);
        border = sh.border;
        if (by_p) {
            z.clear();
            __syncthreads();
        }
    }
    if (by_p) {
        auto bin_left = [=](float v, int i) { return border && st_key(v, i) < border ? -1 : bin_of(v, i); };
        const unsigned q = (unsigned)(border >> ST_IDX_BITS);
        const float least = border ? __uint_as_float((q & 0x80000000u) ? q ^ 0x80000000u : ~q) : -CUDART_INF_F;
        auto cut_left = [=](int bin) { return fmaxf(cut_of(bin), least); };
        if (border) {                                           // of what top-k leaves: few
            z.each(least, [&](float v, int i) {
                const int b = bin_left(v, first + i);
                if (b >= 0) z.add(b, 1, st_weight(v, z.scale, sh.pow2), true);
            });
        } else {                                                // weights of all: those that are far added up in registers
            unsigned n = 0;
            u64 w = 0;
            for (int i = tid * 4; i < z.count; i += THREADS * 4) {
                const float4 v4 = *reinterpret_cast<const float4*>(x + i);
                const float v[4] = {v4.x, v4.y, v4.z, v4.w};
                bool near = false;
                u64 we[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool far = (m - v[e]) * per >= (float)(ST_BINS - 1) && i + e < z.count;      // (bin_of; of two infinities: not)
                    we[e] = st_weight_below(v[e], z.scale, sh.pow2);
                    w += far ? we[e] : 0;
                    n += far ? 1 : 0;
                    near = near || !far;
                }
                if (!near) continue;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < z.count) {
                        const int b = bin_of(v[e], 0);
                        if (b < ST_BINS - 1) z.add(b, 1, v[e] == m ? ST_ONE : we[e], true);
                        else if (!((m - v[e]) * per >= (float)(ST_BINS - 1))) { n++; w += we[e]; }
                    }
            }
            n = __reduce_add_sync(0xffffffffu, n);
            w = st_sum_u64(w);
            if (z.lane == 0 && n) z.add(ST_BINS - 1, n, w, true);      // (a slice's weights are below 2^60: the upper part stays below 2^30)
        }
        z.merge();
        u64 total = 0;
        for (int b = z.lane; b < ST_BINS; b += 32) total += sh.merged[b].weight;
        total = st_sum_u64(total);
        bool more;
        const u64 part = st_times(total, p, more);
        z.select(bin_left, cut_left, true, max(part + (more ? 1 : 0), 1ull));
        border = sh.border;
    }
    // ---- the draw, in the order of the vocabulary: a warp has a run of its own ----
    const unsigned border_order = (unsigned)(border >> ST_IDX_BITS);
    const bool by_min = min_p > 0.f;
    const double least = by_min ? (double)T0 * log((double)fminf(min_p, 1.f)) : 0.;
    float cut = -CUDART_INF_F;                                  // what is below has no part
    if (border) cut = __uint_as_float((border_order & 0x80000000u) ? border_order ^ 0x80000000u : ~border_order);
    if (by_min) cut = fmaxf(cut, __double2float_rd((double)m + least));
    if (!(cut <= m)) cut = m;                                   // (infinities)
    auto weight = [&](float v, int i) -> u64 {
        const unsigned q = st_order(v);
        if (q < border_order || (q == border_order && st_key(v, first + i) < border)) return 0;
        if (by_min && v != m && !((double)v - (double)m >= least)) return 0;
        return st_weight(v, z.scale, sh.pow2);
    };
    auto weights = [&](int i, int end, u64 (&w)[4]) {           // of four neighbours
        w[0] = w[1] = w[2] = w[3] = 0;
        if (i >= end) return;
        const float4 v = *reinterpret_cast<const float4*>(x + i);
        if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= cut)) return;
        w[0] = weight(v.x, i);
        if (i + 1 < end) w[1] = weight(v.y, i + 1);
        if (i + 2 < end) w[2] = weight(v.z, i + 2);
        if (i + 3 < end) w[3] = weight(v.w, i + 3);
    };
    const int run = (a.slice / (THREADS / 32) / 128 + 1) * 128, r0 = z.warp * run, r1 = min(z.count, r0 + run);
    u64 mine = 0;
    for (int i = r0 + z.lane * 4; i < r1; i += 128) {
        u64 w[4];
        weights(i, r1, w);
        mine += (w[0] + w[1]) + (w[2] + w[3]);
    }
    mine = st_sum_u64(mine);
    if (z.lane == 0) sh.warp_sum[z.warp] = mine;
    __syncthreads();
    if (tid < ctas) {
        u64 s = 0;
        for (int w = 0; w < (THREADS / 32); w++) s += sh.warp_sum[w];
        cluster.map_shared_rank(&sh, tid)->cta_sum[rank] = s;
    }
    cluster.sync();
    u64 ahead = 0, total = 0;
    for (int r = 0; r < ctas; r++) {
        if (r < rank) ahead += sh.cta_sum[r];
        total += sh.cta_sum[r];
    }
    const float u = a.coin[row];
    bool more;
    u64 want = u >= 1.f ? total - 1 : u > 0.f ? st_times(total, u, more) : 0;      // the first sum above it
    want = want < total ? want : total - 1;
    for (int w = 0; w < z.warp; w++) ahead += sh.warp_sum[w];
    if (want >= ahead && want < ahead + sh.warp_sum[z.warp]) {
        for (int i0 = r0; i0 < r1; i0 += 128) {
            const int i = i0 + z.lane * 4;
            u64 w[4];
            weights(i, r1, w);
            const u64 s = (w[0] + w[1]) + (w[2] + w[3]);
            u64 incl = s;
#pragma unroll
            for (int o2 = 1; o2 < 32; o2 <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, incl, o2);
                if (z.lane >= o2) incl += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, ahead + incl > want);
            if (hit) {
                if (z.lane == __ffs(hit) - 1) {
                    u64 before = ahead + incl - s;
                    int e = 0;
                    while (e < 3 && before + w[e] <= want) before += w[e++];
                    const float v = x[i + e];
                    a.tokens[row] = first + i + e;
                    if (a.prob != nullptr) a.prob[row] = (float)(exp(v == m ? 0. : ((double)v - (double)m) / (double)T0) * 17592186044416.0 / (double)total);
                }
                break;
            }
            ahead += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
}

extern void dl_set_error(const char* fmt, ...);
extern "C" int dl_device_sm_count();

template <typename T, int THREADS, int PER_SM> static int st_launch(const StArgs& a, int M, int ctas, int pdl, cudaStream_t stream) {
    const size_t smem = sizeof(StShared) + (size_t)a.slice * 4;
    static SmemLimit given;
    auto* kernel = sample_tokens_kernel<T, THREADS, PER_SM>;
    if (const int rc = dl_smem_limit("dl_sample_tokens", kernel, smem, given)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(M * ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
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

// Largest vocabulary of dl_sample_tokens
extern "C" int dl_sample_tokens_max_vocab() { return ST_MAX_CTAS * ST_MAX_SLICE; }

extern "C" int dl_sample_tokens(const void* logits, int type, int M, int vocab, long long ld, const float* temperature, const int* top_k, const float* top_p, const float* min_p, const float* coin,
                                int* tokens_out, float* prob_out, int pdl, void* stream) {
    if (M < 0 || vocab < 1 || vocab > dl_sample_tokens_max_vocab() || M > 1 << 24) { dl_set_error("dl_sample_tokens: %d rows of %d logits (at most %d)", M, vocab, dl_sample_tokens_max_vocab()); return -1; }
    if (ld < vocab && M > 1) { dl_set_error("dl_sample_tokens: rows overlap (ld %lld)", ld); return -1; }
    if (M == 0) return 0;
    if (!logits || !temperature || !coin || !tokens_out) { dl_set_error("dl_sample_tokens: a null pointer"); return -1; }
    int ctas = 1;                                              // 4096 logits a CTA or more
    while (ctas < ST_MAX_CTAS && vocab > ctas * 4096) ctas *= 2;
    const int slice = ((vocab + ctas - 1) / ctas + 31) / 32 * 32;
    const bool wide = ((uintptr_t)logits & 15) == 0 && (M == 1 || ld * (type == 0 ? 4 : 2) % 16 == 0);
    const StArgs a = {logits, ld, temperature, top_p, min_p, coin, top_k, tokens_out, prob_out, vocab, slice, wide ? 1 : 0};
    cudaStream_t st = (cudaStream_t)stream;
    // few rows: an SM for each CTA, and all of its threads
    const bool few = (long long)M * ctas <= dl_device_sm_count();
    if (type == 0) return few ? st_launch<float, 1024, 1>(a, M, ctas, pdl, st) : st_launch<float, 384, 3>(a, M, ctas, pdl, st);
    if (type == 1) return few ? st_launch<__nv_bfloat16, 1024, 1>(a, M, ctas, pdl, st) : st_launch<__nv_bfloat16, 384, 3>(a, M, ctas, pdl, st);
    if (type == 2) return few ? st_launch<__half, 1024, 1>(a, M, ctas, pdl, st) : st_launch<__half, 384, 3>(a, M, ctas, pdl, st);
    dl_set_error("dl_sample_tokens: unsupported type %d", type);
    return -1;
}
