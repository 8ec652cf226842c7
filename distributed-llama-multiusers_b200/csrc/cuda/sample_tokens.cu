// A token for every row of logits from given random numbers: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T); the order of tokens: largest logit first, of equal ones the lowest index first
//   top-k   a token stays if fewer than k are ahead of it;
//   top-p   of those a token stays if the weight ahead of it is below p times the weight of what top-k leaves;
//   min-p   of those a token stays if w_i >= min_p (the largest weight is 1)
//   the token: in the order of the vocabulary the first one where the sum of the weights that stay is above coin times their total
// so what stays is always the front of the order, and one border (logit, index) tells it.  T <= 0: the first of the largest.
//
// A cluster of CTAs per row holds the row's logits in shared memory, read from memory once.  The border is found without sorting: 1024 bins of the distance
// to the maximum with their counts and weights, summed over the cluster, give the bin in which the border lies, and its few tokens are compared with each other.  Where a bin
// holds more than the list takes (logits that are equal, or far below the maximum) it is divided again, by the bits of logit and index together, which
// no two tokens share, until it fits.
//
// Weights are whole numbers of 2^-44, so that sums do not depend on their order; they are exact to 2^-29 of themselves (a table of 64 powers of two and a
// polynomial, after P. T. P. Tang's table-driven exponential, on the difference and the factor as pairs of f32 numbers): with sums of f32 results a
// coin next to a border between two tokens would fall on the other side once in some thousand rows.
#include <math_constants.h>
#include <type_traits>
#include <cuda_bf16.h>
#include "common.cuh"
#include "smem_limit.cuh"

#define ST_THREADS 512
#define ST_WARPS (ST_THREADS / 32)
#define ST_BINS 1024
#define ST_LIST 1024
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
};

struct StSums { u64 weight; u64 count; };

// what the CTAs of a row leave for each other; in each CTA's shared memory
struct StShared {
    unsigned hist[4][ST_BINS];         // counts, and weights in three parts of 15 bits
    u64 list_key[ST_LIST], list_weight[ST_LIST];      // in CTA 0's: the tokens of the border's bin
    StSums merged[ST_BINS];            // this CTA's share of the bins, summed over the cluster
    u64 key[ST_MAX_CTAS];              // each CTA's largest
    StSums total[ST_MAX_CTAS];
    u64 lo[ST_MAX_CTAS], hi[ST_MAX_CTAS];
    StSums above, inside;              // of the bin found: what lies ahead of it and in it
    int bin;
    unsigned listed;
    u64 border, kept;                  // smallest key that stays, weight of what stays
    u64 warp_sum[ST_WARPS];
    u64 cta_sum[ST_MAX_CTAS];
    u64 red[ST_WARPS];
    StSums red2[ST_WARPS];
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

// round(2^44 exp((x - m) / T))
DL_DEVINL u64 st_weight(float x, const StScale& s, const uint2* pow2) {
    if (x == s.m) return ST_ONE;                               // (infinities among them)
    const float d = x - s.m, p = d * s.c_hi;
    if (!(p > -46.f)) return 0;
    const float b = d - x, lost = (x - (d - b)) + (-s.m - b);   // x - m = d + lost
    const float e = fmaf(lost, s.c_hi, fmaf(d, s.c_lo, fmaf(d, s.c_hi, -p)));
    const float t = p + 196608.f;                              // 1.5 2^17: p to the nearest 1 / 64
    const int k = __float_as_int(t) - __float_as_int(196608.f);
    const float r = (p - (t - 196608.f)) + e;                   // at most 2^-7
    const float q = r * fmaf(r, fmaf(r, fmaf(r, 0.00961812911f, 0.0555041087f), 0.240226507f), 0.693147181f);      // 2^r - 1
    const uint2 f = pow2[k & 63];
    const int low = __float_as_int(fmaf(__uint_as_float(f.y), q, 0.046875f)) - __float_as_int(0.046875f);        // 1.5 2^-5: units of 2^-28
    const u64 w = (u64)(f.x + ((unsigned)low << 3)) << 14;
    return ((w >> -(k >> 6)) + 1) >> 1;
}

template <typename T> DL_DEVINL float st_load(const T* p);
template <> DL_DEVINL float st_load<float>(const float* p) { return __ldcs(p); }
template <> DL_DEVINL float st_load<__nv_bfloat16>(const __nv_bfloat16* p) { return __uint_as_float((unsigned)__ldcs(reinterpret_cast<const unsigned short*>(p)) << 16); }
template <> DL_DEVINL float st_load<__half>(const __half* p) { return __half2float(__ushort_as_half(__ldcs(reinterpret_cast<const unsigned short*>(p)))); }

// u f rounded down, and whether something was lost; f in [0, 1)
DL_DEVINL u64 st_times(u64 u, float f, bool& more) {
    const u64 scaled = (u64)((double)f * 9223372036854775808.0) << 1;      // 2^64 f (24 bits of it; below 2^-40 some are lost)
    more = u * scaled != 0;
    return __umul64hi(u, scaled);
}

// The row's work: what all CTAs of its cluster do together.
struct StRow {
    StShared& sh;
    const float* x;
    const int first, count;            // the slice: indexes first .. first + count - 1
    const int rank, ctas, tid, warp, lane;
    cg::cluster_group cluster;
    StScale scale;

    DL_DEVINL StShared* at(int r) const { return cluster.map_shared_rank(&sh, r); }

    // Counts (and weights) of the tokens by bin, summed over the cluster: a share of the bins in each CTA's sh.merged, the shares' sums in sh.total.
    template <typename Bin> DL_DEVINL void histogram(Bin bin_of, bool weights) {
        for (int b = tid; b < 4 * ST_BINS; b += ST_THREADS) (&sh.hist[0][0])[b] = 0;
        __syncthreads();
        for (int i = tid; i < count; i += ST_THREADS) {
            const int b = bin_of(x[i], first + i);
            if (b < 0) continue;
            atomicAdd(&sh.hist[0][b], 1u);
            if (weights) {
                const u64 w = st_weight(x[i], scale, sh.pow2);
                const unsigned w0 = (unsigned)w & 0x7fffu, w1 = (unsigned)(w >> 15) & 0x7fffu, w2 = (unsigned)(w >> 30);
                if (w0) atomicAdd(&sh.hist[1][b], w0);
                if (w1) atomicAdd(&sh.hist[2][b], w1);
                if (w2) atomicAdd(&sh.hist[3][b], w2);
            }
        }
        cluster.sync();
        const int share = ST_BINS / ctas;
        StSums mine = {0, 0};
        for (int b = tid; b < share; b += ST_THREADS) {
            StSums s = {0, 0};
            for (int r = 0; r < ctas; r++) {
                const StShared* o = at(r);
                const int g = rank * share + b;
                s.count += o->hist[0][g];
                s.weight += (u64)o->hist[1][g] + ((u64)o->hist[2][g] << 15) + ((u64)o->hist[3][g] << 30);
            }
            sh.merged[b] = s;
            mine.count += s.count;
            mine.weight += s.weight;
        }
        mine.count = st_sum_u64(mine.count);
        mine.weight = st_sum_u64(mine.weight);
        if (lane == 0) sh.red2[warp] = mine;
        __syncthreads();
        if (tid < ctas) {
            StSums s = {0, 0};
            for (int w = 0; w < ST_WARPS; w++) { s.count += sh.red2[w].count; s.weight += sh.red2[w].weight; }
            at(tid)->total[rank] = s;
        }
        cluster.sync();
    }

    // The bin in which what lies ahead reaches the target (bin 0 is ahead of the others): sh.bin, sh.above, sh.inside in every CTA.
    DL_DEVINL void locate(const StSums& ahead, bool by_weight, u64 target) {
        if (warp == 0) {
            StSums before = ahead;
            bool here = false;
            for (int r = 0; r <= rank; r++) {                  // the crossing lies here if the shares ahead stay below and this one does not
                const StSums t = sh.total[r];
                if (r == rank) here = (by_weight ? before.weight < target && before.weight + t.weight >= target : before.count < target && before.count + t.count >= target);
                else { before.count += t.count; before.weight += t.weight; }
            }
            if (here) {
                const int share = ST_BINS / ctas;
                for (int b0 = 0; b0 < share; b0 += 32) {
                    const StSums s = sh.merged[b0 + lane];
                    StSums incl = s;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const u64 c = __shfl_up_sync(0xffffffffu, incl.count, o), w = __shfl_up_sync(0xffffffffu, incl.weight, o);
                        if (lane >= o) { incl.count += c; incl.weight += w; }
                    }
                    const unsigned hit = __ballot_sync(0xffffffffu, by_weight ? before.weight + incl.weight >= target : before.count + incl.count >= target);
                    if (hit) {
                        if (lane == __ffs(hit) - 1) {
                            const StSums up = {before.weight + incl.weight - s.weight, before.count + incl.count - s.count};
                            for (int r = 0; r < ctas; r++) {
                                StShared* o = at(r);
                                o->bin = rank * share + b0 + lane;
                                o->above = up;
                                o->inside = s;
                            }
                        }
                        break;
                    }
                    before.count += __shfl_sync(0xffffffffu, incl.count, 31);
                    before.weight += __shfl_sync(0xffffffffu, incl.weight, 31);
                }
            }
        }
        cluster.sync();
    }

    // The border for a target: the key of the first token with which the sums reach it.  `bin_of` gave the histogram in place; afterwards sh.border and sh.kept (the
    // weight up to and with that token).  True: the histogram in place is another one now.
    template <typename Bin> DL_DEVINL bool select(Bin bin_of, bool by_weight, u64 target) {
        locate(StSums{0, 0}, by_weight, target);
        StSums above = sh.above, inside = sh.inside;
        int bin = sh.bin;
        u64 lo = 0, hi = ~0ull;                                 // the keys of the bin
        bool range = false;                                    // they are known; `bin` is not looked at any more
        for (int turn = 0; turn < 8 && inside.count > ST_LIST; turn++) {      // (52 bits of key, ten at a time)
            if (!range) {
                u64 least = ~0ull, most = 0;
                for (int i = tid; i < count; i += ST_THREADS)
                    if (bin_of(x[i], first + i) == bin) {
                        const u64 k = st_key(x[i], first + i);
                        least = k < least ? k : least;
                        most = k > most ? k : most;
                    }
                most = st_max_u64(most);
                least = ~st_max_u64(~least);
                if (lane == 0) { sh.red2[warp].weight = most; sh.red2[warp].count = least; }
                __syncthreads();
                if (tid < ctas) {
                    for (int w = 0; w < ST_WARPS; w++) {
                        most = sh.red2[w].weight > most ? sh.red2[w].weight : most;
                        least = sh.red2[w].count < least ? sh.red2[w].count : least;
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
            const int bits = 64 - __clzll(hi - lo), shift = bits > 10 ? bits - 10 : 0;      // (hi > lo: more than one token)
            const u64 top = hi, end = lo;
            histogram([=](float v, int i) { const u64 k = st_key(v, i); return k <= top && k >= end ? (int)((top - k) >> shift) : -1; }, true);
            locate(above, by_weight, target);
            above = sh.above;
            inside = sh.inside;
            hi = top - ((u64)sh.bin << shift);
            const u64 next = hi - ((1ull << shift) - 1);
            lo = hi >= ((1ull << shift) - 1) && next > end ? next : end;
        }
        if (tid == 0 && rank == 0) sh.listed = 0;
        cluster.sync();
        StShared* o = at(0);
        for (int i0 = warp * 32; i0 < count; i0 += ST_THREADS) {
            const int i = i0 + lane;
            u64 k = 0;
            bool mine = i < count;
            if (mine) {
                k = st_key(x[i], first + i);
                mine = range ? k <= hi && k >= lo : bin_of(x[i], first + i) == bin;
            }
            const unsigned any = __ballot_sync(0xffffffffu, mine);
            if (!any) continue;
            unsigned base = 0;
            if (lane == 0) base = atomicAdd(&o->listed, __popc(any));
            base = __shfl_sync(0xffffffffu, base, 0) + __popc(any & ((1u << lane) - 1));
            if (mine && base < ST_LIST) {
                o->list_key[base] = k;
                o->list_weight[base] = st_weight(x[i], scale, sh.pow2);
            }
        }
        cluster.sync();
        if (rank == 0) {
            const int n = (int)min(inside.count, (u64)ST_LIST);
            for (int i = tid; i < n; i += ST_THREADS) {
                const u64 k = sh.list_key[i], w = sh.list_weight[i];
                u64 c = above.count, s = above.weight;
                for (int j = 0; j < n; j++)
                    if (sh.list_key[j] > k) { c++; s += sh.list_weight[j]; }
                if (by_weight ? s < target && s + w >= target : c < target && c + 1 >= target)
                    for (int r = 0; r < ctas; r++) { at(r)->border = k; at(r)->kept = s + w; }
            }
        }
        cluster.sync();
        return range;
    }
};

template <typename T>
__global__ void __launch_bounds__(ST_THREADS, 2) sample_tokens_kernel(const __grid_constant__ StArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    StShared& sh = *reinterpret_cast<StShared*>(smem);
    float* x = reinterpret_cast<float*>(smem + sizeof(StShared));
    const int tid = threadIdx.x;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), row = blockIdx.x / ctas;
    const int first = rank * a.slice;
    StRow z{sh, x, first, max(0, min(a.vocab - first, a.slice)), rank, ctas, tid, tid >> 5, tid & 31, cluster, {0.f, 0.f, 0.f}};
    pdl_launch_dependents();
    if (tid < 64) {
        const double p = exp2((double)tid / 64.0);
        sh.pow2[tid] = make_uint2((unsigned)__double2uint_rn(p * 2147483648.0), __float_as_uint((float)p));
    }
    pdl_wait();
    // ---- the slice into shared memory, and the first of the largest ----
    const T* src = reinterpret_cast<const T*>(a.logits) + (long long)row * a.ld + first;
    u64 best = 0;
#pragma unroll 8
    for (int i = tid; i < z.count; i += ST_THREADS) {
        float v = st_load<T>(src + i);
        v = v == v ? v + 0.f : -CUDART_INF_F;                   // no NaN, no negative zero
        x[i] = v;
        const u64 k = st_key(v, first + i);
        best = k > best ? k : best;
    }
    best = st_max_u64(best);
    if (z.lane == 0) sh.red[z.warp] = best;
    __syncthreads();
    if (tid < ctas) {
        for (int w = 0; w < ST_WARPS; w++) best = sh.red[w] > best ? sh.red[w] : best;
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
    float min_p = a.min_p ? a.min_p[row] : 0.f;
    const bool by_k = k > 0 && k < a.vocab, by_p = p > 0.f && p < 1.f;
    u64 border = 0;
    if (by_k || by_p) {
        // bins of the distance to the maximum: more than ST_REACH below it is the last one (whatever T: the distance is taken in units of it)
        const float per = z.scale.c_hi * (0.69314718f * (ST_BINS - 1) / ST_REACH);
        auto bin_of = [=](float v, int) { return v == m ? 0 : (int)fminf((m - v) * per, (float)(ST_BINS - 1)); };
        z.histogram(bin_of, by_p);
        StSums all = {0, 0};
        for (int r = 0; r < ctas; r++) { all.count += sh.total[r].count; all.weight += sh.total[r].weight; }
        u64 total = all.weight;
        bool divided = false;
        if (by_k) {
            divided = z.select(bin_of, false, (u64)k);
            border = sh.border;
            total = sh.kept;
        }
        if (by_p) {
            if (divided) z.histogram(bin_of, true);
            bool more;
            const u64 part = st_times(total, p, more);
            z.select(bin_of, true, max(part + (more ? 1 : 0), 1ull));
            border = sh.border > border ? sh.border : border;
        }
    }
    // ---- the draw, in the order of the vocabulary: a warp has a run of its own ----
    const unsigned border_order = (unsigned)(border >> ST_IDX_BITS);
    const bool by_min = min_p > 0.f;
    const double least = by_min ? (double)T0 * log((double)fminf(min_p, 1.f)) : 0.;
    auto weight = [&](int i) -> u64 {
        const float v = x[i];
        const unsigned q = st_order(v);
        if (q < border_order || (q == border_order && st_key(v, first + i) < border)) return 0;
        if (by_min && v != m && !((double)v - (double)m >= least)) return 0;
        return st_weight(v, z.scale, sh.pow2);
    };
    const int run = (a.slice / ST_WARPS + 31) / 32 * 32, r0 = z.warp * run, r1 = min(z.count, r0 + run);
    u64 mine = 0;
    for (int i = r0 + z.lane; i < r1; i += 32) mine += weight(i);
    mine = st_sum_u64(mine);
    if (z.lane == 0) sh.warp_sum[z.warp] = mine;
    __syncthreads();
    if (tid < ctas) {
        u64 s = 0;
        for (int w = 0; w < ST_WARPS; w++) s += sh.warp_sum[w];
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
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + z.lane;
            const u64 w = i < r1 ? weight(i) : 0;
            u64 incl = w;
#pragma unroll
            for (int o2 = 1; o2 < 32; o2 <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, incl, o2);
                if (z.lane >= o2) incl += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, ahead + incl > want);
            if (hit) {
                if (z.lane == __ffs(hit) - 1) {
                    a.tokens[row] = first + i;
                    if (a.prob != nullptr) a.prob[row] = (float)(exp(x[i] == m ? 0. : ((double)x[i] - (double)m) / (double)T0) * 17592186044416.0 / (double)total);
                }
                break;
            }
            ahead += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
}

extern void dl_set_error(const char* fmt, ...);

template <typename T> static int st_launch(const StArgs& a, int M, int ctas, int pdl, cudaStream_t stream) {
    const size_t smem = sizeof(StShared) + (size_t)a.slice * 4;
    static SmemLimit given;
    if (const int rc = dl_smem_limit("dl_sample_tokens", sample_tokens_kernel<T>, smem, given)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(M * ctas));
    cfg.blockDim = dim3(ST_THREADS);
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T>, a);
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
    const StArgs a = {logits, ld, temperature, top_p, min_p, coin, top_k, tokens_out, prob_out, vocab, slice};
    cudaStream_t st = (cudaStream_t)stream;
    if (type == 0) return st_launch<float>(a, M, ctas, pdl, st);
    if (type == 1) return st_launch<__nv_bfloat16>(a, M, ctas, pdl, st);
    if (type == 2) return st_launch<__half>(a, M, ctas, pdl, st);
    dl_set_error("dl_sample_tokens: unsupported type %d", type);
    return -1;
}
