// What the attention kernels on tcgen05 have in common (attention_prefill_tc.cu, shared_attention.cu): tensor-memory copies, softmax weights from scores in
// registers, the two products' MMAs on 128-byte-swizzled tiles of 128 rows, waits that end.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"
#include "f32_pairs.cuh"

DL_DEVINL void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
DL_DEVINL void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
DL_DEVINL void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
// instruction descriptor, kind::f16: A fp16 / bf16 K-major (or TMEM), B alike with selectable major-ness, D f32
DL_DEVINL uint32_t pt_idesc(int M, int N, int b_mn_major, bool bf16) {
    uint32_t d = 0;
    d |= 1u << 4;                                  // D = f32
    if (bf16) d |= (1u << 7) | (1u << 10);         // A and B = bf16
    d |= (uint32_t)(b_mn_major & 1) << 16;         // b_major: 0 = K, 1 = MN
    d |= (uint32_t)(N >> 3) << 17;
    d |= (uint32_t)(M >> 4) << 24;
    return d;
}
DL_DEVINL float pt_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool NAN_TOO> DL_DEVINL float pt_max(float a, float b) {      // NAN_TOO: of a NaN and a number the NaN
    if (!NAN_TOO) return fmaxf(a, b);
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
template <bool LINES> DL_DEVINL uint32_t pt_pack2(float lo, float hi) {
    if (LINES) {
        __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

// exp2 on the FMA pipe (Cody-Waite split + degree-3 polynomial, relative error 8e-5 -- the result is rounded to fp16,
// 5e-4, right after; LINES, whose other kernels form it in full: degree 5, 2e-7): the softmax is bound by the 16 MUFU results
// per clock and SM (128 x 128 exp2 per step = 1024 clk, as long as the MMAs of the step), so every fourth element takes this
// path instead
template <bool LINES> DL_DEVINL pair_f pt_ex2_poly(pair_f x) {
    float lo, hi;                                  // LINES: a NaN stays one, as in the mma.sync kernel
    pair_get(x, lo, hi);
    if (LINES) {
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(-126.0f));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(-126.0f));
    } else {
        lo = fmaxf(lo, -126.0f);
        hi = fmaxf(hi, -126.0f);
    }
    auto both = [](float c) { return pair_of(c, c); };
    const pair_f xc = pair_of(lo, hi), t = add2(xc, both(12582912.0f));                 // 1.5 * 2^23: round(x) lands in the low mantissa bits
    const pair_f f = fma2(add2(t, both(-12582912.0f)), both(-1.0f), xc);                // [-0.5, 0.5]
    float tl, th, pl, ph;
    pair_get(t, tl, th);
    if (LINES) {
        const pair_f p = fma2(fma2(fma2(fma2(fma2(both(1.32764725e-3f), f, both(9.67554096e-3f)), f, both(0.0555071309f)), f, both(0.240221202f)), f, both(0.693146944f)), f, both(1.00000012f));
        return mul2(p, pair_of(__int_as_float((__float_as_int(tl) << 23) + 0x3f800000), __int_as_float((__float_as_int(th) << 23) + 0x3f800000)));
    }
    pair_get(fma2(fma2(fma2(both(0.0550886838f), f, both(0.242604051f)), f, both(0.693276242f)), f, both(0.99992894f)), pl, ph);
    return pair_of(__int_as_float(__float_as_int(pl) + (__float_as_int(tl) << 23)), __int_as_float(__float_as_int(ph) + (__float_as_int(th) << 23)));
}

// 32 scores (masked ones are -inf) -> exp2(s * sc - ref) as 16 packed fp16 pairs; their sum is added to `sum`.  LINES: as bf16 and, in `lo`, the
// bf16 remainder of each, 17 bits together
template <bool LINES> DL_DEVINL void pt_probs(const uint32_t (&v)[32], float sc, float ref, uint32_t (&pk)[16], uint32_t (&lo)[LINES ? 16 : 1], pair_f& sum) {
    const pair_f sc2 = pair_of(sc, sc), ref2 = pair_of(-ref, -ref);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
        pair_f p = fma2(pair_of(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc2, ref2);
        float pa, pb;
        if ((e & 6) == 6) {
            p = pt_ex2_poly<LINES>(p);
            pair_get(p, pa, pb);
        } else {
            pair_get(p, pa, pb);
            pa = pt_ex2(pa);
            pb = pt_ex2(pb);
            p = pair_of(pa, pb);
        }
        sum = add2(sum, p);
        pk[e >> 1] = pt_pack2<LINES>(pa, pb);
        if constexpr (LINES) lo[e >> 1] = pt_pack2<LINES>(pa - __uint_as_float(pk[e >> 1] << 16), pb - __uint_as_float(pk[e >> 1] & 0xffff0000u));
    }
}

// The eight MMAs of a group (K = 128) by one thread of the converged warp, elected by a predicate: with one MMA at a time inside an `if (elect)`
// 4001 rows of 32 heads took 150 us, 138 so (on the same inputs again and again, with the queries loaded by warps of their own).
// D += A B^T, both operands 128-byte-swizzled half tiles 16 KB apart (32 B of a row per MMA)
DL_DEVINL void pt_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t.reg .b32 x, y;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|p, 0xffffffff;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.eq.b32 r, 0, 0;\n\t"
        "add.u32 x, %1, 0; add.u32 y, %2, 0; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, q;\n\t"
        "add.u32 x, %1, 2; add.u32 y, %2, 2; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 4; add.u32 y, %2, 4; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 6; add.u32 y, %2, 6; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 1024; add.u32 y, %2, 1024; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 1026; add.u32 y, %2, 1026; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 1028; add.u32 y, %2, 1028; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 1030; add.u32 y, %2, 1030; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// ... of heads of 64: the first half tiles alone
DL_DEVINL void pt_mma_ss4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t.reg .b32 x, y;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|p, 0xffffffff;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.eq.b32 r, 0, 0;\n\t"
        "add.u32 x, %1, 0; add.u32 y, %2, 0; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, q;\n\t"
        "add.u32 x, %1, 2; add.u32 y, %2, 2; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 4; add.u32 y, %2, 4; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t"
        "add.u32 x, %1, 6; add.u32 y, %2, 6; mov.b64 a, {x, %3}; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, r;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D += A B, A in tensor memory (8 columns per MMA), B MN-major (two 8-token groups of 1024 B per MMA)
DL_DEVINL void pt_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t.reg .b32 x, y;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|p, 0xffffffff;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.eq.b32 r, 0, 0;\n\t"
        "add.u32 x, %1, 0; add.u32 y, %2, 0; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, q;\n\t"
        "add.u32 x, %1, 8; add.u32 y, %2, 128; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t"
        "add.u32 x, %1, 16; add.u32 y, %2, 256; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t"
        "add.u32 x, %1, 24; add.u32 y, %2, 384; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t"
        "add.u32 x, %1, 32; add.u32 y, %2, 512; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t"
        "add.u32 x, %1, 40; add.u32 y, %2, 640; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t"
        "add.u32 x, %1, 48; add.u32 y, %2, 768; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t"
        "add.u32 x, %1, 56; add.u32 y, %2, 896; mov.b64 b, {y, %3}; @p tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, r;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
DL_DEVINL void pt_commit(uint64_t* bar) {
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}

// A wait that gives up (the CTA has had its time, WAIT_DEADLINE_NS): the flag ends the other waits, too, every output of the CTA becomes a NaN, and
// the host learns of it by dl_attention_status()
struct PtWaits {
    volatile int* gave_up;
    unsigned long long t0, ns;
    DL_DEVINL void operator()(uint64_t* bar, uint32_t parity) const {
        unsigned n = 0;
        while (!mbar_try_wait(bar, parity)) {
            if ((++n & 0x3FFu) == 0) {
                if (*gave_up) return;
                if (globaltimer_ns() - t0 > ns) { *gave_up = 1; return; }
            }
        }
    }
};
