// Attention over a paged 4-bit cache for requests with many rows (queries times query heads a kv head): the same
// function as kv4_attend.cu, on the 5th-generation tensor cores.
//
// A CTA takes a tile of 256 rows of a (request, kv head) (128 at D = 256) and walks its keys in steps of 128 (64 at
// D = 256). Per step
//   * the codes of its keys and values become fp16 tiles in shared memory, (code | 1024) - 1024 and one fused multiply-add
//     with the group's scale and bias (times a power of two), pairs (i, i + 4) of a word as they come out of one mask. The
//     order of dimensions that this makes is met by the queries (stored in the same order) and undone when the output is
//     written;
//   * one thread issues S = Q K^T (both in shared memory, K-major) and O += P V (P in tensor memory, V in shared memory as
//     it lies, dimensions contiguous: the transposed B operand) as tcgen05.mma with fp32 accumulators in tensor memory:
//     for two query tiles in turn, S0 PV0 S1 PV1 ..., so that one tile's softmax runs beside the other's products;
//   * each of 256 threads owns a row: it reads its scores, keeps the running maximum and sum in fp32, and writes its
//     probabilities back over them as fp16. The row's output is only rescaled when its maximum has grown by 2^8; until then a
//     step is one pass over the scores (`once`), its probabilities in registers. (Both are published methods.)
// Two forms, by how often a key is met again (pf_dense):
//   * unpacked in place: eight warps unpack, one step ahead through registers, told by a page warp where the keys lie; the
//     registers of the block are shared out by role (setmaxnreg);
//   * DENSE: kv4_dense_kernel unpacks the keys and values of such requests once, to tiles in the workspace as they are to
//     lie in shared memory, and one thread copies them in whole (cp.async.bulk). Unpacking beside the products costs both:
//     128 keys at D = 128 take 1.45 us of products alone, 1.29 of unpacking alone, 2.5 together.
// Roundings to fp16: queries after a power of two a row (exact for bf16 but for values 2^-26 below the row's largest); keys,
// values and probabilities, 2^-11 each against the 2^-8 of a bf16 output (an fp16 output's error against 64 bits grows by
// them from 2.1e-4 to 2.4e-4 .. 4.6e-4 of its size, mostly by the keys': the tensor cores take the operands in no finer type
// but at half the rate). Keys after a power of two a step that puts the largest that its groups can hold at 2^14 .. 2^15, taken back with the
// scores' factor: a group's scale and a sixteenth of it stay normal numbers down to 2^-20 of that, where the group's share of
// a score is as small. Values after a power of two a step in the same way; a row's outputs have one of their own, and its
// probabilities are multiplied by the difference while that is small, its outputs (as its maximum's growth does) where it
// is not: so a step's values cost another step's no bits, and a row only those of the keys that it sees. A step with keys, or
// keys' values, that are 2^-20 of the largest or less has one a key (PF_WILD; key_exp), which each row's scores or probabilities
// take in, in a step of two passes: the large ones may be out of a row's sight. Within a key, values are held to 2^-31 of its
// largest, and probabilities to 2^-31 of the row's largest.
// A masked score is -inf, its probability 0; a value whose scale or bias is not finite is held as 0 and its key as NaN,
// so that only rows that see it become NaN.
// Work is dealt out as in kv4_attend.cu: the steps of all tiles (each as far as its last row sees) evenly over one CTA a
// SM, parts joined by kv4_prefill_join_kernel.
// What bounds it: 4 D operations a row and key on the tensor cores, and one exponential a row and key at 16 a clock and SM,
// which take as long as the products do at D = 128 (tensor pipe 47% busy, exponentials 47%: they are not yet beside each
// other all the time). Measured, GPU time of a call, bf16: 4,096 new tokens on 28,672 cached, 16 heads on 2, D = 128: 1,086 to
// 1,153 us = 894 to 949 TFLOP/s by the clock that the power limit leaves (55 to 58% of the measured peak), fp16 1,218 to 1,276;
// a mixed batch of 8 (1 to 1,024 new on up to 2,048 cached, 32 heads on 8): 194 us = 494 TFLOP/s, the items' ends and short
// tiles; 16 requests of 5 drafted tokens on up to 4,003 keys, 16 heads on 2, D = 256: 52 to 54 us, latency: 4 us to find the
// share, 6 to fetch the queries, 2 to 8 steps, 2 to write, and the joins. The powers of two a step, row and key take 3 to 5% of
// these, and 9% of the drafts and of the fp16 piece.
// Tried and slower: half the exponentials as polynomials (1,128 against 1,081 us); 4 unpacking warps of 128 registers (1,778);
// the two-pass step out of line (a mixed batch 245 against 200); a row's powers of two in shared memory (no faster);
// 48 registers for the issuing warp (1,904); query rows fetched by neighbouring lanes (no faster, and 1,061 against 1,029).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "kv4_attend.cuh"
#include "lq_host.h"
#include "lq_ptx.cuh"
#include "lq_status.cuh"

namespace lq {

constexpr int PF_SOFT = 8;                       // softmax warps (a row a thread)
constexpr int PF_UNPACK = 8;                     // unpacking warps
constexpr int PF_FIRST = 4;                      // the first warpgroup: an issuing warp, one for pages or copies, two idle
// Threads a CTA: without unpacking warps 168 registers each, with them 96 each at launch, then shared out.
constexpr int pf_threads(bool dense) { return (PF_FIRST + PF_SOFT + (dense ? 0 : PF_UNPACK)) * 32; }
constexpr int PF_REGS_SOFT = 120, PF_REGS_UNPACK = 88, PF_REGS_MMA = 64;
static_assert(PF_SOFT * PF_REGS_SOFT + PF_UNPACK * PF_REGS_UNPACK + PF_FIRST * PF_REGS_MMA <= pf_threads(false) / 32 * 96, "registers");

template <int D>
struct PfShape {
    static constexpr int GR = D / 64;
    static constexpr int NQ = D == 256 ? 1 : 2;   // query tiles of 128 rows
    static constexpr int R = 128 * NQ;
    static constexpr int KT = D == 256 ? 64 : 128;  // keys a step
    static constexpr int RB = D / 2;
    static constexpr int QB = 128 * D * 2;        // bytes of a query tile
    static constexpr int TB = KT * D * 2;         // bytes of a key (or value) tile
    static constexpr int SLAB = KT * 128;         // bytes of 64 dimensions of a tile
    static constexpr int SMEM = NQ * QB + 4 * TB; // + barriers
    static constexpr int O_COL = 2 * KT;          // tensor memory: two score buffers, then the outputs
    static_assert(2 * KT + NQ * D <= 512, "tensor memory columns");
};

// What an item costs beside its steps (queries fetched, the pipeline filled, outputs written), in steps. A mixed batch of 8:
// 4: 177.5 us, 5: 175.8, 7: 179.4.
constexpr int PF_ITEM = 5;

// A tile's steps of keys: from the first that its first row sees to the last that its last row sees.
template <int D>
__device__ __forceinline__ void pf_steps(const Kv4AttArgs& a, int base, int fresh, int tile, int* lo, int* hi) {
    using S = PfShape<D>;
    const int room = int(min((long long)a.width * a.pool.page, 0x7fffffffLL));
    const int q0 = tile * S::R / a.G, q1 = (min((tile + 1) * S::R, fresh * a.G) - 1) / a.G;
    const int keys = max(min(base + q1 + 1, room), 0);
    const int from = a.window ? min(max(base + q0 + 1 - a.window, 0), keys) : 0;
    *lo = min(from, max(keys - 1, 0)) / S::KT;
    *hi = max((keys + S::KT - 1) / S::KT, *lo + 1);
}

template <int D>
__device__ __forceinline__ int pf_tiles(const Kv4AttArgs& a, int b, int* first, int* fresh, int* base) {
    const Kv4Req r = kv4_new(a, b);
    *first = r.first;
    *fresh = r.fresh;
    *base = r.len - r.fresh;
    return r.fresh * a.G > a.split_rows ? (r.fresh * a.G + PfShape<D>::R - 1) / PfShape<D>::R : 0;
}

// Units of every `step`-th of request b's tiles, from tile `from` on.
template <int D>
__device__ __forceinline__ long long pf_weight(const Kv4AttArgs& a, int b, int from, int step) {
    int first, fresh, base;
    const int tiles = pf_tiles<D>(a, b, &first, &fresh, &base);
    long long w = 0;
    for (int t = from; t < tiles; t += step) {
        int lo, hi;
        pf_steps<D>(a, base, fresh, t, &lo, &hi);
        w += hi - lo + PF_ITEM;
    }
    return w * a.pool.KVH;
}

// Inclusive sum over the CTA's threads, and their total.
__device__ __forceinline__ long long pf_scan(long long v, long long* red, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    __syncthreads();  // (red may still be read from before)
    if (lane == 31) red[warp] = v;
    __syncthreads();
    long long sum = 0;
    for (int k = 0; k < int(blockDim.x >> 5); ++k) {
        if (k == warp) v += sum;
        sum += red[k];
    }
    *total = sum;
    return v;
}

// The CTA's walk over its share: items (request, tile, kv head) in that order, each with its steps [st0, st1). A share is
// counted in units: PF_ITEM of each item, then its steps.
template <int D>
struct PfWalk {
    int left, skip;  // units of the share left; units of the next item that come before the share
    bool begun;
    int b, tile, kvh, lo, hi, st0, st1, first, fresh, base, tiles;

    // The next item with a step in the share; false when the share is done. Every caller walks alike.
    __device__ bool next(const Kv4AttArgs& a) {
        while (left) {
            if (begun && ++kvh == a.pool.KVH) {
                kvh = 0;
                if (++tile >= tiles) {
                    do {
                        ++b;
                        tiles = pf_tiles<D>(a, b, &first, &fresh, &base);
                    } while (!tiles);
                    tile = 0;
                }
                pf_steps<D>(a, base, fresh, tile, &lo, &hi);
            }
            begun = true;
            const int end = min(hi - lo + PF_ITEM, skip + left);
            st0 = max(skip - PF_ITEM, 0);
            st1 = max(end - PF_ITEM, 0);
            left -= end - skip;
            skip = 0;
            if (st0 < st1) return true;
        }
        return false;
    }
};

__device__ __forceinline__ void pf_tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ void pf_tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// tc_mma_f16 and tc_mma_ts with the operands' places as constant offsets from a tile's, put together inside: kept as values,
// the descriptors of all products would take more registers than the issuing thread has, and each reload delays a product.
template <int A_OFF, int B_OFF, int ACC>
__device__ __forceinline__ void pf_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\t"
        "add.u32 x, %1, %5;\n\tadd.u32 y, %2, %6;\n\t"
        "mov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "n"(A_OFF), "n"(B_OFF), "n"(ACC)
        : "memory");
}
template <int A_OFF, int B_OFF>
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 x, y;\n\t.reg .b64 db;\n\t"
        "add.u32 x, %1, %5;\n\tadd.u32 y, %2, %6;\n\t"
        "mov.b64 db, {y, %3};\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "n"(A_OFF), "n"(B_OFF), "r"(accumulate)
        : "memory");
}
// S (128 rows x KT keys) = Q K^T over the D dimensions, 16 at a time.
template <int D, int SLAB, int... I>
__device__ __forceinline__ void pf_scores(uint32_t d, uint32_t q, uint32_t k, uint32_t hi, uint32_t idesc,
                                          std::integer_sequence<int, I...>) {
    (pf_mma_ss<((I >> 2) * 16384 + (I & 3) * 32) / 16, ((I >> 2) * SLAB + (I & 3) * 32) / 16, (I > 0)>(d, q, k, hi, idesc), ...);
}
// O (128 rows x D) (+)= P V over the step's keys, 16 at a time.
template <int... I>
__device__ __forceinline__ void pf_products(uint32_t d, uint32_t p, uint32_t v, uint32_t hi, uint32_t idesc, uint32_t first,
                                            std::integer_sequence<int, I...>) {
    (pf_mma_ts<I * 8, I * 2048 / 16>(d, p, v, hi, idesc, I > 0 ? 1u : first), ...);
}

// Two 32-bit floats at a time.
__device__ __forceinline__ uint64_t pf_pair(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void pf_unpair(uint64_t v, float* lo, float* hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(v));
}
__device__ __forceinline__ uint64_t pf_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pf_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// What a pair of probabilities adds to its row's sum. fp16 outputs: as they were rounded, so that what a rounding adds to a
// row's weights is divided out again (a row that sees one key is that key's value); for bf16 outputs it is too little to matter.
template <typename T>
__device__ __forceinline__ void pf_summand(uint32_t h, float* e0, float* e1) {
    if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        *e0 = f.x, *e1 = f.y;
    }
}

// Descriptor of a B operand whose N side is contiguous (128-byte swizzle): 8 keys of 64 dimensions are 1024 bytes, the
// next 8 keys follow (stride offset), the next 64 dimensions lie a slab away (leading offset).
__device__ __forceinline__ uint64_t pf_desc_v(uint32_t addr, uint32_t slab) {
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(slab >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// (v - 1024) * s + b on fp16 pairs: v - 1024 exact, the rest rounded once.
__device__ __forceinline__ uint32_t pf_affine(uint32_t v, uint32_t s2, uint32_t b2) {
    const uint32_t magic = 0x64006400u;
    const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&magic));
    const __half2 r = __hfma2(q, *reinterpret_cast<const __half2*>(&s2), *reinterpret_cast<const __half2*>(&b2));
    return *reinterpret_cast<const uint32_t*>(&r);
}

struct PfBars {
    uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2], r_full[4], r_empty[4], done;
    int abort;          // a wait gave up: no one waits any more
    int exps[4];        // powers of two of the keys and values of step i & 3 (pf_exps)
    uint32_t miss[4];   // its runs of 8 keys without a page
    alignas(16) int8_t key_exp[4][256];  // powers of two of its keys' values, and (from KT on) of the keys, where they differ
                                         // widely (PF_WILD)
    // what the page warp tells the unpacking warps of step i & 3: the pool row of each run of 8 keys (none: KV4_NONE), the
    // keys from its first to the tile's end (0: no more steps), and the runs without a page
    uint32_t run[4][16];
    int left[4];
    uint32_t gone[4];
    float k_max[2][PF_UNPACK], v_max[2][PF_UNPACK];  // of step i & 1: what each unpacking warp's groups can hold at most
    float k_min[2][PF_UNPACK], v_min[2][PF_UNPACK];  // (values: negative from a warp that has no step), and the least of that
    int rows, steps;    // the item's (0: no more), from the first softmax warp to the issuing thread
};

// A bounded wait that, once any has given up, none of the CTA's takes again. After that every role still comes to its end by
// itself: what it computes is void, but no warp waits at a barrier that another has passed by. Warps that meet at a barrier
// (the unpacking ones, and the lanes of the page warp) leave their loops only together, on a word that all of them read
// after they met; the others meet no one before the end. Copies and products in flight are waited for before the CTA ends.
__device__ __forceinline__ void pf_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (*abort) return;
    if (!mbar_wait(bar, parity)) *abort = 1;
}

// Which keys and which 16 bytes of codes piece j of a lane of warp uw (of W) is: 8 lanes are 8 keys, so that their stores
// fall on different banks.
template <int D, int W>
struct PfPieces {
    static constexpr int NP = D / 32, J = PfShape<D>::KT * NP / (W * 32);  // pieces a key, a lane
    __device__ static __forceinline__ int key(int j, int uw, int lane) {
        const int blk = j * W + uw;
        return NP == 2 ? blk * 16 + (lane & 7) + ((lane >> 4) << 3) : NP == 4 ? blk * 8 + (lane & 7) : (blk >> 1) * 8 + (lane & 7);
    }
    __device__ static __forceinline__ int piece(int j, int uw, int lane) {
        return NP == 2 ? (lane >> 3) & 1 : NP == 4 ? lane >> 3 : (lane >> 3) + 4 * ((j * W + uw) & 1);
    }
};

// 32 codes with one scale and bias -> 64 bytes of a tile row (128-byte swizzle), 16 bytes at a time.
template <int D>
__device__ __forceinline__ void pf_unpack(const uint4& codes, float s, float b, uint32_t tile, int key, int p) {
    const uint32_t s1 = cvt_f16x2(s, s), s16 = cvt_f16x2(s * 0.0625f, s * 0.0625f), b2 = cvt_f16x2(b, b);
    const uint32_t cw[4] = {codes.x, codes.y, codes.z, codes.w};
    const uint32_t row = tile + (p >> 1) * PfShape<D>::SLAB + key * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = cw[i], y = cw[i] >> 8;
        const uint32_t o0 = pf_affine(lop3_and_or(x, 0x000f000fu, 0x64006400u), s1, b2);
        const uint32_t o1 = pf_affine(lop3_and_or(x, 0x00f000f0u, 0x64006400u), s16, b2);
        const uint32_t o2 = pf_affine(lop3_and_or(y, 0x000f000fu, 0x64006400u), s1, b2);
        const uint32_t o3 = pf_affine(lop3_and_or(y, 0x00f000f0u, 0x64006400u), s16, b2);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + ((((p & 1) * 4 + i) ^ (key & 7)) << 4)), "r"(o0), "r"(o1),
                     "r"(o2), "r"(o3)
                     : "memory");
    }
}

// (Down to 2^-20 of a step's largest, a value's rounding and its scales' are below 2^-11. What holds less than PF_LEAST is not
// asked for: groups and tokens of zeros, to which the quantizer gives scales of 1e-7.)
constexpr float PF_LEAST = 0x1p-19f;
__device__ __forceinline__ bool pf_wild(float least, float most) { return least < most * 0x1p-20f; }

// A piece's scales and biases in fp32. A value scale or bias that is not finite makes the values 0 and the key NaN, which
// only the rows that see it meet; so does an infinite key. Adds the largest |key| and |value| that the groups can hold, and
// the least of them (from PF_LEAST on).
template <typename T>
__device__ __forceinline__ void pf_scales(uint16_t ks16, uint16_t kb16, uint16_t vs16, uint16_t vb16, float* ks, float* kb,
                                          float* vs, float* vb, float* k_top, float* v_top, float* k_low, float* v_low) {
    *ks = F16Traits<T>::to_f32(ks16), *kb = F16Traits<T>::to_f32(kb16);
    *vs = F16Traits<T>::to_f32(vs16), *vb = F16Traits<T>::to_f32(vb16);
    const float k_most = fmaf(15.0f, fabsf(*ks), fabsf(*kb)), v_most = fmaf(15.0f, fabsf(*vs), fabsf(*vb));
    if (!(v_most < INFINITY)) {
        *vs = *vb = 0.0f;
        *ks = *kb = __int_as_float(0x7fffffff);
        return;
    }
    *v_top = fmaxf(*v_top, v_most);
    if (v_most >= PF_LEAST) *v_low = fminf(*v_low, v_most);
    if (k_most < INFINITY) {
        *k_top = fmaxf(*k_top, k_most);
        if (k_most >= PF_LEAST) *k_low = fminf(*k_low, k_most);
    }
}
// 2^e, e in -126 .. 127.
__device__ __forceinline__ float pf_pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
// The power of two that puts M at 2^14 .. 2^15 (at least -113; 0 for 0).
__device__ __forceinline__ int pf_fit(float M) { return M > 0.0f ? min(14 - (int(__float_as_uint(M) >> 23) - 127), 110) : 0; }
// The powers of two of a step's keys and values in one word.
__device__ __forceinline__ int pf_exps(int ke, int ve) { return int(uint32_t(ke) << 16 | (uint32_t(ve) & 0xffffu)); }
// The values' of a step (or key) that holds none but zeros: any; and of a step whose keys, and their values, have one each.
constexpr int PF_ANY = 127, PF_WILD = 126;
__device__ __forceinline__ int8_t pf_key_exp(int top) { return int8_t(top ? pf_fit(__int_as_float(top)) : PF_ANY); }
// A key's largest (or its values') from its groups' that are finite (the bits of floats from 0 on are in their order).
__device__ __forceinline__ void pf_key_max(int* top, float s, float b) {
    const float most = fmaf(15.0f, fabsf(s), fabsf(b));
    if (most < INFINITY) atomicMax(top, __float_as_int(most));
}
// Whether keys differ so widely, and not only a key's groups (a head of 64 dimensions in a place of 128): asked of whole warps.
template <int KT>
__device__ __forceinline__ bool pf_wild_keys(const int* top, float most) {
    unsigned least = 0x7f800000u;
#pragma unroll
    for (int k = threadIdx.x & 31; k < KT; k += 32) {
        const unsigned x = unsigned(*reinterpret_cast<const volatile int*>(top + k));
        if (x >= unsigned(__float_as_uint(PF_LEAST))) least = min(least, x);
    }
    return pf_wild(__uint_as_float(__reduce_min_sync(0xffffffffu, least)), most);
}
// Probabilities are held 2^PF_BIAS times as large, so that fp16 has those down to 2^-20 of the row's largest in full, and
// 2^-31 of it at least. Their upper end leaves room for a maximum that has grown by 2^PF_LAG since the row's reference and for
// outputs that lie 2^PF_UP from a step's values, 2^15 in all; 2^PF_DOWN costs small ones bits, of values that are as much smaller.
// Beyond these a row gets a new reference or power of two, which takes the step's scores twice (PF_LAG 5: a mixed batch 231 us
// against 192).
constexpr int PF_BIAS = 6, PF_LAG = 8, PF_UP = 1, PF_DOWN = -4;  // (a power of two of values is at most 110)

// ---- the dense form's first pass: the keys and values of requests with many tiles, unpacked once ----
// One CTA a (step of KT keys, kv head, request): the step's two tiles as they are to lie in shared memory, copied out whole,
// and its keys' and values' powers of two and missing pages.
constexpr int PD_WARPS = 8;
template <typename T, int D>
__global__ void __launch_bounds__(PD_WARPS * 32) kv4_dense_kernel(const Kv4AttArgs a) {
    using S = PfShape<D>;
    using P = PfPieces<D, PD_WARPS>;
    extern __shared__ __align__(1024) uint8_t pf_raw[];
    __shared__ float part[PD_WARPS], k_part[PD_WARPS], low_part[PD_WARPS], k_low_part[PD_WARPS];
    __shared__ int key_top[2][S::KT];  // of the values, of the keys
    grid_dep_wait();
    const int s = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int first, fresh, base, lo, hi;
    if (!pf_tiles<D>(a, b, &first, &fresh, &base)) return;
    pf_steps<D>(a, base, fresh, 0, &lo, &hi);
    const int room = int(min((long long)a.width * a.pool.page, 0x7fffffffLL)), keys = max(min(base + fresh, room), 0);
    if (s < lo || s >= max((keys + S::KT - 1) / S::KT, 1)) return;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pf_raw) + 127) & ~uintptr_t(127));
    const uint32_t tile = smem_u32(smem);
    constexpr int RUNS = S::KT / 8;
    const int seen_from = a.window ? max(base + 1 - a.window, 0) : 0;  // (the first query's)
    const int key0 = s * S::KT, run_key = key0 + (lane % RUNS) * 8;
    uint32_t mine = KV4_NONE;
    bool gone = false;
    if (run_key < keys && run_key + 8 > seen_from) {  // (what lies behind a window may have been freed)
        const int pg = run_key / a.pool.page, id = a.table[(size_t)b * a.width + pg];
        gone = unsigned(id) >= unsigned(a.pool.pages);
        if (gone)
            record_status(LQ_DEV_BOUNDS);
        else
            mine = kv4_row(a.pool, id, kvh, run_key - pg * a.pool.page);
    }
    const uint32_t miss = __ballot_sync(0xffffffffu, lane < RUNS && gone);
    uint4 kc[P::J], vc[P::J];
    float ks[P::J], kb[P::J], vs[P::J], vb[P::J], k_top = 0.0f, top = 0.0f, k_low = INFINITY, low = INFINITY;
    uint16_t sc[P::J][4];
#pragma unroll
    for (int j = 0; j < P::J; ++j) {
        const int k = P::key(j, warp, lane), p = P::piece(j, warp, lane);
        const uint32_t run = __shfl_sync(0xffffffffu, mine, k / 8);
        kc[j] = vc[j] = make_uint4(0, 0, 0, 0);
        sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0;
        if (run != KV4_NONE && key0 + k < keys) {
            const size_t row = run + (k & 7), g = row * S::GR + p / 2;
            kc[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.pool.kq) + row * S::RB + p * 16);
            vc[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.pool.vq) + row * S::RB + p * 16);
            sc[j][0] = a.pool.ks[g], sc[j][1] = a.pool.kb[g], sc[j][2] = a.pool.vs[g], sc[j][3] = a.pool.vb[g];
        }
    }
#pragma unroll
    for (int j = 0; j < P::J; ++j)
        pf_scales<T>(sc[j][0], sc[j][1], sc[j][2], sc[j][3], &ks[j], &kb[j], &vs[j], &vb[j], &k_top, &top, &k_low, &low);
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    k_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(k_top)));
    low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low)));
    k_low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(k_low)));
    if (lane == 0) part[warp] = top, k_part[warp] = k_top, low_part[warp] = low, k_low_part[warp] = k_low;
    if (threadIdx.x < S::KT) key_top[0][threadIdx.x] = key_top[1][threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PD_WARPS; ++i) {
        top = fmaxf(top, part[i]), k_top = fmaxf(k_top, k_part[i]);
        low = fminf(low, low_part[i]), k_low = fminf(k_low, k_low_part[i]);
    }
    const size_t at = ((size_t)b * a.pool.KVH + kvh) * a.dense_steps + s;
    bool wild = pf_wild(low, top) || pf_wild(k_low, k_top);
    if (wild) {
#pragma unroll
        for (int j = 0; j < P::J; ++j) {
            pf_key_max(&key_top[0][P::key(j, warp, lane)], vs[j], vb[j]);
            pf_key_max(&key_top[1][P::key(j, warp, lane)], ks[j], kb[j]);
        }
        __syncthreads();
        wild = pf_wild_keys<S::KT>(key_top[0], top) || pf_wild_keys<S::KT>(key_top[1], k_top);
        if (wild && threadIdx.x < 2 * S::KT)
            a.dense_keys[at * (2 * S::KT) + threadIdx.x] = pf_key_exp(key_top[threadIdx.x / S::KT][threadIdx.x % S::KT]);
    }
    const int ke = pf_fit(k_top);
    const float kf = pf_pow2(ke);
    const int ve = pf_fit(top);
    const float vf = pf_pow2(ve);
#pragma unroll
    for (int j = 0; j < P::J; ++j) {
        const int k = P::key(j, warp, lane), p = P::piece(j, warp, lane);
        const float f = wild ? pf_pow2(pf_fit(__int_as_float(key_top[0][k]))) : vf;
        const float fk = wild ? pf_pow2(pf_fit(__int_as_float(key_top[1][k]))) : kf;
        pf_unpack<D>(kc[j], ks[j] * fk, kb[j] * fk, tile, k, p);
        pf_unpack<D>(vc[j], vs[j] * f, vb[j] * f, tile + S::TB, k, p);
    }
    fence_proxy_async();
    __syncthreads();
    if (threadIdx.x == 0) {
        a.dense_meta[at] = make_int2(pf_exps(ke, wild ? PF_WILD : top > 0.0f ? ve : PF_ANY), int(miss));
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.dense + at * (2 * S::TB)), "r"(tile),
                     "r"(2 * S::TB)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
    }
}

// What a row sees of keys 32 i .. 32 i + 31 of a step, a bit a key: [lo, hi) of the step's keys but for its missing runs.
__device__ __forceinline__ uint32_t pf_sees(int lo, int hi, uint32_t miss, int i) {
    const int from = min(max(lo - 32 * i, 0), 32), to = min(max(hi - 32 * i, 0), 32);
    uint32_t v = uint32_t((1ull << to) - 1) & ~uint32_t((1ull << from) - 1);
    const uint32_t gone = (miss >> (4 * i)) & 15;
    if (gone) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((gone >> k) & 1) v &= ~(0xffu << (8 * k));
    }
    return v;
}
__device__ __forceinline__ float pf_seen(uint32_t score, uint32_t v, int i) { return (v >> i) & 1 ? __uint_as_float(score) : -INFINITY; }
// The scores' factor (a positive number, so that a masked score stays -inf).
__device__ __forceinline__ float pf_factor(float c, int exps) {
    return fminf(fmaxf(c * pf_pow2(-(exps >> 16)), 1.17549435e-38f), 3.4028234e38f);
}

// A row's running maximum (base 2) and sum, its outputs' power of two, and the least of the steps' that this was fitted to.
struct PfRow {
    float m, l;
    int ve, ve_low;
};

// A new maximum mn, and, of a step that gives one (sized), a new power of two of the outputs: the step's, but no more than 2^64
// above the least of the steps' before, whose sums (below 2^50) then stay within 32 bits' range. Returns what the outputs are
// multiplied by.
__device__ __forceinline__ float pf_refit(PfRow& row, float mn, int ve_t, bool sized) {
    int to = row.ve;
    if (sized) row.ve_low = min(row.ve_low, ve_t), to = min(ve_t, row.ve_low + 64);
    const float decay = mn > row.m ? kv4_ex2(row.m - mn) : 1.0f;
    const float corr = row.m == -INFINITY ? 0.0f : decay * pf_pow2(max(to - row.ve, -126));
    row.l *= decay;
    row.m = mn;
    row.ve = to;
    return corr;
}

// A row's step whose keys and values have powers of two each (PF_WILD), in two passes over its scores (s_col), which its
// probabilities replace; before: products into its outputs (o_col) so far, 0 for none. Out of line, since it is rare.
template <typename T, int D>
__device__ __noinline__ PfRow pf_wild_step(PfRow row, PfBars* bars, int it, int w, int before, uint32_t s_col, uint32_t o_col,
                                            int lo, int hi, float c) {
    constexpr int KT = PfShape<D>::KT;
    const uint32_t miss = *reinterpret_cast<volatile uint32_t*>(&bars->miss[it & 3]), key_exp = smem_u32(bars->key_exp[it & 3]);
    auto factor = [&](uint32_t k) {  // of a key's score, from the word that holds its power of two in the low byte
        const int ke = int8_t(k);
        return pf_factor(c, ke == PF_ANY ? 0 : ke * 65536);
    };
    int ve_t = PF_ANY;  // the largest values' that the row sees
#pragma unroll 1
    for (int k = 0; k < KT; k += 4) {
        const uint32_t v = pf_sees(lo, hi, miss, k / 32) >> (k & 31), x = lds32(key_exp + k);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((v >> i) & 1) ve_t = min(ve_t, int(int8_t(x >> (8 * i))));
    }
    const bool sized = ve_t != PF_ANY;
    if (!sized) ve_t = row.ve;
    float mx = -INFINITY;
#pragma unroll 1
    for (int ch = 0; ch < KT / 32; ++ch) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(s_col + ch * 32, r);
        const uint32_t v = pf_sees(lo, hi, miss, ch);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const uint32_t k = lds32(key_exp + KT + ch * 32 + (i & ~3)) >> (8 * (i & 2));
            mx = fmaxf(fmaxf(mx, pf_seen(r[i], v, i) * factor(k)), pf_seen(r[i + 1], v, i + 1) * factor(k >> 8));
        }
    }
    const float mn = fmaxf(row.m, mx);
    const bool some = mx != -INFINITY;
    const int d = row.ve - ve_t;
    const bool grow = mn > row.m + PF_LAG || (row.m == -INFINITY && mn > row.m) || (some && (d < PF_DOWN || d > PF_UP));
    if (__any_sync(0xffffffffu, grow)) {
        const float corr = pf_refit(row, mn, ve_t, some && sized);
        if (before) {
            pf_wait(&bars->o_done[w], (before - 1) & 1, &bars->abort);  // the last product is in
            tc_fence_after();
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(o_col + ch * 32, r);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
                tmem_st_32x32b_x32(o_col + ch * 32, r);
            }
        }
    }
    const float mz = row.m == -INFINITY ? 0.0f : row.m;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int ch = 0; ch < KT / 16; ++ch) {
        uint32_t x[16], p[8];
        tmem_ld_32x32b_x16(s_col + ch * 16, x);
        const uint32_t v = pf_sees(lo, hi, miss, ch >> 1) >> (16 * (ch & 1));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint32_t kk = lds32(key_exp + KT + ch * 16 + (i & ~3)) >> (8 * (i & 2));
            const float e0 = kv4_ex2(fmaf(pf_seen(x[i], v, i), factor(kk), -mz));
            const float e1 = kv4_ex2(fmaf(pf_seen(x[i + 1], v, i + 1), factor(kk >> 8), -mz));
            // (the small ones' may become 0 beside the large ones')
            const uint32_t k = lds32(key_exp + ch * 16 + (i & ~3)) >> (8 * (i & 2));
            p[i / 2] = cvt_f16x2(e1 * pf_pow2(min(max(row.ve - int(int8_t(k >> 8)) + PF_BIAS, -126), 100)),
                                 e0 * pf_pow2(min(max(row.ve - int(int8_t(k)) + PF_BIAS, -126), 100)));
            sum[i & 2] += e0;
            sum[(i & 2) + 1] += e1;
        }
        pf_tmem_st8(s_col + ch * 8, p);
    }
    row.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    return row;
}

// DENSE: the tiles come unpacked, by bulk copies, from what kv4_dense_kernel left.
template <typename T, int D, bool DENSE>
__global__ void __launch_bounds__(pf_threads(DENSE), 1) kv4_prefill_kernel(const Kv4AttArgs a) {
    using S = PfShape<D>;
    constexpr int GR = S::GR, KT = S::KT, NQ = S::NQ, R = S::R, PF_THREADS = pf_threads(DENSE);
    extern __shared__ __align__(1024) uint8_t pf_raw[];
    __shared__ long long red[PF_THREADS / 32];
    __shared__ uint8_t* volatile pf_base;
    __shared__ int key_top[DENSE ? 1 : KT];  // bits of the largest that a key's groups can hold, while those are found
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (smem_u32(pf_raw) & 1023) {  // (the declaration's alignment; there is no room to make up for it)
        if (tid == 0) record_status(LQ_DEV_BOUNDS);
        return;
    }
    if (tid == 0) {
        uint8_t* smem = pf_raw;
        PfBars& bar = *reinterpret_cast<PfBars*>(smem + S::SMEM);
        pf_base = smem;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.q_full[i], 4);
            mbar_init(&bar.k_full[i], DENSE ? 1 : PF_UNPACK);
            mbar_init(&bar.k_empty[i], 1);
            mbar_init(&bar.v_full[i], DENSE ? 1 : PF_UNPACK);
            mbar_init(&bar.v_empty[i], 1);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 4);
            mbar_init(&bar.o_done[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar.r_full[i], 1);
            mbar_init(&bar.r_empty[i], PF_UNPACK);
        }
        mbar_init(&bar.done, 1);
        bar.abort = 0;
        fence_barrier_init();
    }
    grid_dep_wait();
    if (a.split_rows == 0) kv4_zero_rest(a, D);  // (else kv4_attend does)
    // ---- this CTA's share ----
    // up to 32 threads a request sum its tiles' units; then requests, and the tiles of the one found, are scanned together
    int each = 32;
    while (each > 1 && a.B * each > PF_THREADS) each >>= 1;
    const int round = PF_THREADS / each;
    auto weight = [&](int b0) -> long long {  // (in the first of a request's threads)
        const int b = b0 + tid / each, from = tid & (each - 1);
        long long w = b < a.B ? pf_weight<D>(a, b, from, each) : 0;
        for (int d = 1; d < each; d <<= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
        return from ? 0 : w;
    };
    __shared__ long long found_at;
    __shared__ int found;
    long long sum0, total;
    const long long w0 = weight(0), s0 = pf_scan(w0, red, &sum0);
    total = sum0;
    for (int b0 = round; b0 < a.B; b0 += round) {
        long long sum;
        pf_scan(weight(b0), red, &sum);
        total += sum;
    }
    const int n = int(min((long long)gridDim.x, total));
    int32_t* rec = a.records + blockIdx.x * 8;  // what the join kernel does for this CTA's first step
    if (int(blockIdx.x) >= n) {
        if (tid == 0) rec[0] = 0;
        return;
    }
    const long long x0 = (long long)blockIdx.x * total / n, x1 = ((long long)blockIdx.x + 1) * total / n;
    PfWalk<D> walk;
    long long item;
    {
        long long at = 0;
        for (int b0 = 0;; b0 += round) {
            long long w = w0, s = s0, sum = sum0;
            if (b0) {
                w = weight(b0);
                s = pf_scan(w, red, &sum);
            }
            if (at + sum <= x0) {
                at += sum;
                continue;
            }
            if (at + s > x0 && at + s - w <= x0) found = b0 + tid / each, found_at = at + s - w;  // one thread's
            __syncthreads();
            walk.b = found;
            at = found_at;
            break;
        }
        walk.tiles = pf_tiles<D>(a, walk.b, &walk.first, &walk.fresh, &walk.base);
        walk.tile = 0;
        for (int t0 = 0; walk.tiles > 1; t0 += PF_THREADS) {
            int lo = 0, hi = 0;
            if (t0 + tid < walk.tiles) pf_steps<D>(a, walk.base, walk.fresh, t0 + tid, &lo, &hi);
            const long long w = t0 + tid < walk.tiles ? (long long)(hi - lo + PF_ITEM) * a.pool.KVH : 0;
            long long sum;
            const long long s = pf_scan(w, red, &sum);
            if (at + sum <= x0) {
                at += sum;
                continue;
            }
            if (at + s > x0 && at + s - w <= x0) found = t0 + tid, found_at = at + s - w;
            __syncthreads();
            walk.tile = found;
            at = found_at;
            break;
        }
        pf_steps<D>(a, walk.base, walk.fresh, walk.tile, &walk.lo, &walk.hi);
        const int units = walk.hi - walk.lo + PF_ITEM;
        walk.kvh = int((x0 - at) / units);
        item = at + (long long)walk.kvh * units;
        walk.skip = int(x0 - item);
        walk.left = int(x1 - x0);
        walk.begun = false;
    }

    __shared__ uint32_t tmem_base;
    if (warp == 0) {
        tmem_alloc(&tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid == 64) {  // (an idle warp's)
        const int c0 = kv4_owner(item + PF_ITEM, total, n), c1 = kv4_owner(item + walk.hi - walk.lo + PF_ITEM - 1, total, n);
        rec[0] = walk.skip > PF_ITEM && c0 == int(blockIdx.x) - 1;  // the first boundary within its item's steps
        rec[1] = walk.first;
        rec[2] = walk.tile * R;
        rec[3] = min(R, walk.fresh * a.G - walk.tile * R);
        rec[4] = walk.kvh;
        rec[5] = c1;
    }
    // Each role reads the bases for itself from here on: values shared by all roles would be kept on the stack by all,
    // those with registers to spare too, and the issuing thread's reloads would delay its products.
    struct Places {
        PfBars& bar;
        volatile int* abort;
        uint32_t tmem, sq, sk, sv;
    };
    auto places = [&]() -> Places {
        uint8_t* smem = pf_base;
        PfBars& bar = *reinterpret_cast<PfBars*>(smem + S::SMEM);
        const uint32_t sq = smem_u32(smem), sk = sq + NQ * S::QB;
        return {bar, &bar.abort, *reinterpret_cast<volatile uint32_t*>(&tmem_base), sq, sk, sk + 2 * S::TB};
    };
    const int room = int(min((long long)a.width * a.pool.page, 0x7fffffffLL));

    if (warp >= PF_FIRST && warp < PF_FIRST + PF_SOFT) {
        // ------------------------------ softmax: a row a thread ------------------------------
        if constexpr (!DENSE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PF_REGS_SOFT));
        const Places at = places();
        PfBars& bar = at.bar;
        volatile int* const abort = at.abort;
        const uint32_t tmem = at.tmem, sq = at.sq;
        const int w = (warp - PF_FIRST) >> 2, wr = (warp & 3) * 32 + lane;  // query tile, row in it
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        int it = 0, used = 0;  // steps of the CTA, and of this query tile
        while (walk.next(a)) {
            const int row0 = walk.tile * R, rows = min(R, walk.fresh * a.G - row0);
            const int steps = walk.st1 - walk.st0;
            if (w * 128 >= rows || w >= NQ) {  // no rows here
                it += steps;
                continue;
            }
            const int row = w * 128 + wr;
            const bool live = row < rows;
            const int rr = row0 + (live ? row : rows - 1), qi = rr / a.G, head = walk.kvh * a.G + rr - qi * a.G;
            const int row_hi = min(walk.base + qi + 1, room);
            const int row_lo = a.window ? max(walk.base + qi + 1 - a.window, 0) : 0;
            if (walk.base + walk.fresh > room) record_status(LQ_DEV_BOUNDS);
            // the warp's rows all see [lo_all, hi_all)
            const int hi_all = __reduce_min_sync(0xffffffffu, row_hi), lo_all = __reduce_max_sync(0xffffffffu, row_lo);

            // the query row, a power of two larger, in the order of the unpacked codes
            const size_t qo = ((size_t)(walk.first + qi) * a.H + head) * D;
            float c;
            {
                const uint4* src = reinterpret_cast<const uint4*>(a.q + qo);
                constexpr int NV = D == 256 ? 16 : D / 8;  // 16-byte pieces held at a time
                const bool some = live && a.scale_log2 != 0.0f;
                uint4 raw[NV];
                float mx = 0.0f;
#pragma unroll
                for (int h = 0; h < D / 8; h += NV) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) raw[i] = some ? src[h + i] : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mx = fmaxf(mx, fmaxf(fabsf(F16Traits<T>::to_f32(x[k] & 0xffffu)),
                                                 fabsf(F16Traits<T>::to_f32(x[k] >> 16))));
                    }
                }
                int E = mx > 0.0f ? 12 - (int((__float_as_uint(mx) >> 23) & 0xff) - 127) : 0;
                E = min(E, 126);  // (from -116, an infinity's)
                const float f = some ? copysignf(__uint_as_float(uint32_t(127 + E) << 23), a.scale_log2) : 0.0f;
                c = a.scale_log2 != 0.0f ? fabsf(a.scale_log2) * __uint_as_float(uint32_t(127 - E) << 23) : 1.0f;
                const uint32_t dst = sq + w * S::QB + wr * 128;
#pragma unroll
                for (int h = 0; h < D / 8; h += NV) {
                    if (D / 8 > NV) {
#pragma unroll
                        for (int i = 0; i < NV; ++i) raw[i] = some ? src[h + i] : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                        float q[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            q[2 * k] = F16Traits<T>::to_f32(x[k] & 0xffffu) * f;
                            q[2 * k + 1] = F16Traits<T>::to_f32(x[k] >> 16) * f;
                        }
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + ((h + i) >> 3) * 16384 + (((i & 7) ^ (wr & 7)) << 4)),
                                     "r"(cvt_f16x2(q[4], q[0])), "r"(cvt_f16x2(q[5], q[1])), "r"(cvt_f16x2(q[6], q[2])),
                                     "r"(cvt_f16x2(q[7], q[3]))
                                     : "memory");
                    }
                }
            }
            if (warp == PF_FIRST && lane == 0) bar.rows = rows, bar.steps = steps;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.q_full[w]);

            PfRow row_at = {-INFINITY, 0.0f, 0, 1000};
            const uint32_t o_col = tmem + lanes + S::O_COL + w * D;
            for (int t = 0; t < steps; ++t, ++it, ++used) {
                const int buf = NQ == 2 ? w : used & 1;
                const uint32_t par = NQ == 2 ? used & 1 : (used >> 1) & 1;
                pf_wait(&bar.s_full[buf], par, abort);
                tc_fence_after();
                const int key0 = (walk.lo + walk.st0 + t) * KT;
                const uint32_t miss = *reinterpret_cast<volatile uint32_t*>(&bar.miss[it & 3]);
                // How far the row's outputs lie from the step's values: its probabilities are multiplied by 2^that. (Below PF_DOWN
                // for PF_WILD. Read where it is used: the one pass needs the registers.)
                auto exps = [&]() { return *reinterpret_cast<volatile int*>(&bar.exps[it & 3]); };
                auto apart = [&]() {
                    const int ve_t = int16_t(exps());
                    return ve_t == PF_ANY ? 0 : row_at.ve - ve_t;
                };
                const bool all = key0 >= lo_all && key0 + KT <= hi_all && miss == 0;
                const uint32_t s_col = tmem + lanes + buf * KT;
                // One query tile: a step's scores are issued before the last step's product, so that without this a warp could
                // be done with an item while two products are to come, and the barrier's parity would take the one before both
                // for the last. Before this step's probabilities are given out, the next product cannot be mistaken.
                auto settled = [&]() {
                    if (NQ == 1 && used > 0) pf_wait(&bar.o_done[w], (used - 1) & 1, abort);
                };
                // The common case, one pass: the reference from the steps before serves the step (found out at its end: the
                // probabilities stay in registers until then, the scores in place).
                auto once = [&](auto masked) -> bool {
                    const float ct = pf_factor(c, exps()), md = float(apart() + PF_BIAS) - row_at.m;
                    const uint64_t c2 = pf_pair(ct, ct), m2 = pf_pair(md, md);
                    constexpr int CH = 16;  // scores at a time (32: 1082 against 1040 us for a 4096-token prompt piece)
                    uint32_t r[2][CH], p[KT / 2];
                    uint64_t sums[2] = {0, 0};
                    float mx[2] = {-INFINITY, -INFINITY};
                    uint32_t v = 0;
                    tmem_ld_32x32b_x16(s_col, r[0]);
#pragma unroll
                    for (int ch = 0; ch < KT / CH; ++ch) {  // the next scores are read while these are worked on
                        uint32_t(&x)[CH] = r[ch & 1];
                        tmem_wait_ld();
                        if (ch + 1 < KT / CH) tmem_ld_32x32b_x16(s_col + (ch + 1) * CH, r[(ch + 1) & 1]);
                        if constexpr (decltype(masked)::value) v = ch & 1 ? v >> 16 : pf_sees(row_lo - key0, row_hi - key0, miss, ch / 2);
#pragma unroll
                        for (int i = 0; i < CH; i += 2) {
                            float s0 = __uint_as_float(x[i]), s1 = __uint_as_float(x[i + 1]);
                            if constexpr (decltype(masked)::value) s0 = pf_seen(x[i], v, i), s1 = pf_seen(x[i + 1], v, i + 1);
                            mx[(i >> 1) & 1] = fmaxf(fmaxf(mx[(i >> 1) & 1], s0), s1);
                            float e0, e1;
                            pf_unpair(pf_fma2(pf_pair(s0, s1), c2, m2), &e0, &e1);
                            e0 = kv4_ex2(e0);
                            e1 = kv4_ex2(e1);
                            const uint32_t h = cvt_f16x2(e1, e0);
                            pf_summand<T>(h, &e0, &e1);
                            sums[(i >> 1) & 1] = pf_add2(sums[(i >> 1) & 1], pf_pair(e0, e1));
                            p[(ch * CH + i) / 2] = h;
                        }
                    }
                    if (__any_sync(0xffffffffu, fmaxf(mx[0], mx[1]) * ct > row_at.m + PF_LAG)) return false;
#pragma unroll
                    for (int ch = 0; ch < KT / 64; ++ch) pf_tmem_st32(s_col + ch * 32, &p[ch * 32]);
                    float a0, a1, b0, b1;
                    pf_unpair(sums[0], &a0, &a1);
                    pf_unpair(sums[1], &b0, &b1);
                    row_at.l = fmaf((a0 + a1) + (b0 + b1), pf_pow2(-apart() - PF_BIAS), row_at.l);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    settled();
                    if (lane == 0) mbar_arrive(&bar.p_full[buf]);
                    return true;
                };
                if (__all_sync(0xffffffffu, row_at.m != -INFINITY && unsigned(apart() - PF_DOWN) <= unsigned(PF_UP - PF_DOWN))) {
                    if (all ? once(std::false_type()) : once(std::true_type())) continue;
                }
                // A new reference (an item's first step, mostly): two passes, in loops, since their code is not often in reach.
                int ve_t = int16_t(exps());
                if (ve_t == PF_WILD) {
                    row_at = pf_wild_step<T, D>(row_at, &bar, it, w, t > 0 ? used : 0, s_col, o_col, row_lo - key0, row_hi - key0, c);
                } else {
                    const float ct = pf_factor(c, exps());
                    const bool sized = ve_t != PF_ANY;
                    if (!sized) ve_t = row_at.ve;
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int ch = 0; ch < KT / 32; ++ch) {
                        uint32_t r[32];
                        tmem_ld_32x32b_x32(s_col + ch * 32, r);
                        const uint32_t v = pf_sees(row_lo - key0, row_hi - key0, miss, ch);
                        tmem_wait_ld();
                        float part[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            part[(i >> 1) & 1] = fmaxf(fmaxf(part[(i >> 1) & 1], pf_seen(r[i], v, i)), pf_seen(r[i + 1], v, i + 1));
                        mx = fmaxf(mx, fmaxf(part[0], part[1]));
                    }
                    const float mn = fmaxf(row_at.m, mx * ct);
                    const bool some = mx != -INFINITY;
                    const int d = row_at.ve - ve_t;
                    const bool grow = mn > row_at.m + PF_LAG || (row_at.m == -INFINITY && mn > row_at.m) || (some && (d < PF_DOWN || d > PF_UP));
                    if (__any_sync(0xffffffffu, grow)) {
                        const float corr = pf_refit(row_at, mn, ve_t, some && sized);
                        if (t > 0) {
                            pf_wait(&bar.o_done[w], (used - 1) & 1, abort);  // the last product is in
                            tc_fence_after();
#pragma unroll 1
                            for (int ch = 0; ch < D / 32; ++ch) {
                                uint32_t r[32];
                                tmem_ld_32x32b_x32(o_col + ch * 32, r);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
                                tmem_st_32x32b_x32(o_col + ch * 32, r);
                            }
                        }
                    }
                    // (below PF_DOWN only after so large values that this step's are nothing beside them: their probabilities are 0
                    // in fp16, and still in the row's sum; and beyond PF_UP only in rows that see nothing of the step)
                    const int dd = min(max(row_at.ve - ve_t, -60), 60) + PF_BIAS;
                    const float mz = (row_at.m == -INFINITY ? 0.0f : row_at.m) - float(dd);
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                    for (int ch = 0; ch < KT / 16; ++ch) {
                        uint32_t x[16], p[8];
                        tmem_ld_32x32b_x16(s_col + ch * 16, x);
                        const uint32_t v = pf_sees(row_lo - key0, row_hi - key0, miss, ch >> 1) >> (16 * (ch & 1));
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float e0 = kv4_ex2(fmaf(pf_seen(x[i], v, i), ct, -mz));
                            float e1 = kv4_ex2(fmaf(pf_seen(x[i + 1], v, i + 1), ct, -mz));
                            p[i / 2] = cvt_f16x2(e1, e0);
                            pf_summand<T>(p[i / 2], &e0, &e1);
                            sum[i & 2] += e0;
                            sum[(i & 2) + 1] += e1;
                        }
                        pf_tmem_st8(s_col + ch * 8, p);
                    }
                    row_at.l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), pf_pow2(-dd), row_at.l);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                settled();
                if (lane == 0) mbar_arrive(&bar.p_full[buf]);
            }
            // ---- the row's output ----
            pf_wait(&bar.o_done[w], (used - 1) & 1, abort);
            tc_fence_after();
            const bool whole = walk.st0 == 0 && walk.st1 == walk.hi - walk.lo;
            const size_t part = ((size_t)blockIdx.x * 2 + (walk.st0 == 0 ? 1 : 0)) * R + row;
            const float m = row_at.m, l = row_at.l, back = pf_pow2(-row_at.ve - PF_BIAS);
            float f = back;
            if (whole) {
                const float sink = kv4_sink(a.sinks, head), M = fmaxf(m, sink);
                const float L = M == -INFINITY ? l : l * kv4_ex2(m - M) + kv4_ex2(sink - M);
                f = L == 0.0f ? 0.0f : back * (M == -INFINITY ? 1.0f : kv4_ex2(m - M)) / L;
            } else if (live) {
                a.part_ml[2 * part] = m;
                a.part_ml[2 * part + 1] = l;
            }
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(o_col + ch * 32, r);
                tmem_wait_ld();
                if (!live) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v[8];  // back in order: place 2 j holds dimension j, place 2 j + 1 dimension j + 4
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[j] = __uint_as_float(r[8 * k + 2 * j]) * f;
                        v[j + 4] = __uint_as_float(r[8 * k + 2 * j + 1]) * f;
                    }
                    if (whole) {
                        uint4 o;
                        o.x = F16Traits<T>::pack2(v[1], v[0]), o.y = F16Traits<T>::pack2(v[3], v[2]);
                        o.z = F16Traits<T>::pack2(v[5], v[4]), o.w = F16Traits<T>::pack2(v[7], v[6]);
                        *reinterpret_cast<uint4*>(a.out + qo + ch * 32 + k * 8) = o;
                    } else {
                        float4* dst = reinterpret_cast<float4*>(a.part_o + part * D + ch * 32 + k * 8);
                        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
            }
            tc_fence_before();
        }
        if (w == 0) {  // no more items
            if (warp == PF_FIRST && lane == 0) bar.rows = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.q_full[0]);
        }
    } else if (warp >= PF_FIRST) {
        if constexpr (!DENSE) {
        // ------------------------------ codes to fp16 tiles ------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PF_REGS_UNPACK));
        const Places at = places();
        PfBars& bar = at.bar;
        volatile int* const abort = at.abort;
        const uint32_t sk = at.sk, sv = at.sv;
        const int uw = warp - PF_FIRST - PF_SOFT;
        using P = PfPieces<D, PF_UNPACK>;
        constexpr int J = P::J;
        // A step's codes, scales and biases in registers.
        struct Held {
            uint4 k[J], v[J];
            uint16_t ks[J], kb[J], vs[J], vb[J];
        };
        int asked = 0;
        // issues the next step's loads; false (for the whole warp) when there is none
        auto fetch = [&](Held& h) -> bool {
            const int slot = asked & 3;
            pf_wait(&bar.r_full[slot], (asked >> 2) & 1, abort);
            const int left = *reinterpret_cast<volatile int*>(&bar.left[slot]);
            if (__any_sync(0xffffffffu, left == 0 || *abort)) return false;
            ++asked;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int k = P::key(j, uw, lane), p = P::piece(j, uw, lane);
                const uint32_t run = *reinterpret_cast<volatile uint32_t*>(&bar.run[slot][k / 8]);
                h.k[j] = h.v[j] = make_uint4(0, 0, 0, 0);
                h.ks[j] = h.kb[j] = h.vs[j] = h.vb[j] = 0;
                if (run != KV4_NONE && k < left) {
                    const size_t row = run + (k & 7), g = row * GR + p / 2;
                    h.k[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.pool.kq) + row * S::RB + p * 16);
                    h.v[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.pool.vq) + row * S::RB + p * 16);
                    h.ks[j] = a.pool.ks[g], h.kb[j] = a.pool.kb[g], h.vs[j] = a.pool.vs[g], h.vb[j] = a.pool.vb[g];
                }
            }
            return true;
        };
        // one step from its registers to the tiles; false, in all warps at the same step, once one of them has none (at the
        // end, or after an error, which they need not see at the same step)
        auto step_out = [&](const Held& h, int it, bool have) -> bool {
            const int st = it & 1;
            const uint32_t par = ((it >> 1) & 1) ^ 1;
            float k_top = 0.0f, top = 0.0f, k_low = INFINITY, low = INFINITY, ks[J], kb[J], vs[J], vb[J];
            if (have) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    pf_scales<T>(h.ks[j], h.kb[j], h.vs[j], h.vb[j], &ks[j], &kb[j], &vs[j], &vb[j], &k_top, &top, &k_low, &low);
            }
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
            k_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(k_top)));
            low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low)));
            k_low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(k_low)));
            if (lane == 0) {
                bar.v_max[st][uw] = have ? top : -1.0f, bar.k_max[st][uw] = k_top;
                bar.v_min[st][uw] = low, bar.k_min[st][uw] = k_low;
            }
            __syncwarp();
            // (a slot is written again after the next step's barrier, which its readers pass later)
            named_barrier(1, PF_UNPACK * 32);
            float M = 0.0f;
            bool over = false;
#pragma unroll
            for (int i = 0; i < PF_UNPACK; ++i) {
                const float x = reinterpret_cast<volatile float*>(bar.v_max[st])[i];
                M = fmaxf(M, x);
                k_top = fmaxf(k_top, reinterpret_cast<volatile float*>(bar.k_max[st])[i]);
                low = fminf(low, reinterpret_cast<volatile float*>(bar.v_min[st])[i]);
                k_low = fminf(k_low, reinterpret_cast<volatile float*>(bar.k_min[st])[i]);
                over = over || x < 0.0f;
            }
            if (over) return false;
            const int ke = pf_fit(k_top);
            const float kf = pf_pow2(ke);
            const int ve = pf_fit(M);
            const float vf = pf_pow2(ve);
            bool wild = pf_wild(low, M) || pf_wild(k_low, k_top);  // (the same in all warps)
            int8_t* const key_exp = bar.key_exp[it & 3];
            if (wild) {
                const int me = uw * 32 + lane;
                wild = false;
#pragma unroll
                for (int keys = 0; keys < 2; ++keys) {  // values, keys
                    if (me < KT) key_top[me] = 0;
                    __syncwarp();
                    named_barrier(1, PF_UNPACK * 32);
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        pf_key_max(&key_top[P::key(j, uw, lane)], keys ? ks[j] : vs[j], keys ? kb[j] : vb[j]);
                    __syncwarp();
                    named_barrier(1, PF_UNPACK * 32);
                    wild = pf_wild_keys<KT>(key_top, keys ? k_top : M) || wild;
                    if (me < KT) key_exp[keys * KT + me] = pf_key_exp(key_top[me]);
                    __syncwarp();
                    named_barrier(1, PF_UNPACK * 32);
                }
            }
            // A key's own: of its values, or (from KT on) of itself.
            auto own = [&](int key) -> float {
                const int e = *reinterpret_cast<volatile int8_t*>(key_exp + key);
                return pf_pow2(e == PF_ANY ? 0 : e);
            };
            if (uw == 0 && lane == 0) {
                bar.exps[it & 3] = pf_exps(ke, wild ? PF_WILD : M > 0.0f ? ve : PF_ANY);
                bar.miss[it & 3] = bar.gone[it & 3];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.r_empty[it & 3]);
            pf_wait(&bar.k_empty[st], par, abort);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float f = wild ? own(KT + P::key(j, uw, lane)) : kf;
                pf_unpack<D>(h.k[j], ks[j] * f, kb[j] * f, sk + st * S::TB, P::key(j, uw, lane), P::piece(j, uw, lane));
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.k_full[st]);
            pf_wait(&bar.v_empty[st], par, abort);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float f = wild ? own(P::key(j, uw, lane)) : vf;
                pf_unpack<D>(h.v[j], vs[j] * f, vb[j] * f, sv + st * S::TB, P::key(j, uw, lane), P::piece(j, uw, lane));
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.v_full[st]);
            return true;
        };
        // two steps a turn, so that what is in flight stays in its registers
        Held h0, h1;
        bool first = fetch(h0);
        for (int it = 0;; it += 2) {
            const bool second = first && fetch(h1);
            if (!step_out(h0, it, first)) break;
            first = second && fetch(h0);
            if (!step_out(h1, it + 1, second)) break;
        }
        }
    } else {
        if constexpr (!DENSE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PF_REGS_MMA));
    }
    if (DENSE && warp == 1) {
        // ------------------------------ copies of the unpacked tiles: one thread ------------------------------
        if (lane == 0) {
            const Places at = places();
            PfBars& bar = at.bar;
            volatile int* const abort = at.abort;
            const uint32_t sk = at.sk, sv = at.sv;
            auto copy = [&](uint64_t* full, uint32_t dst, const void* src, uint32_t bytes) {
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                             "l"(src), "r"(bytes), "r"(smem_u32(full))
                             : "memory");
            };
            int it = 0, keys = 0, values = 0;  // steps, copies
            while (walk.next(a) && !*abort) {
                const size_t tile0 = ((size_t)walk.b * a.pool.KVH + walk.kvh) * a.dense_steps + walk.lo;
                for (int t = walk.st0; t < walk.st1; ++t, ++it) {
                    const int st = it & 1;
                    const uint32_t par = ((it >> 1) & 1) ^ 1;
                    const int2 meta = a.dense_meta[tile0 + t];
                    const uint8_t* src = a.dense + (tile0 + t) * (2 * S::TB);
                    pf_wait(&bar.k_empty[st], par, abort);
                    if (*abort) break;
                    bar.exps[it & 3] = meta.x;
                    bar.miss[it & 3] = uint32_t(meta.y);
                    const bool wild = int16_t(meta.x) == PF_WILD;
                    mbar_arrive_expect_tx(&bar.k_full[st], wild ? S::TB + 2 * KT : S::TB);
                    copy(&bar.k_full[st], sk + st * S::TB, src, S::TB);
                    if (wild) copy(&bar.k_full[st], smem_u32(bar.key_exp[it & 3]), a.dense_keys + (tile0 + t) * (2 * KT), 2 * KT);
                    ++keys;
                    pf_wait(&bar.v_empty[st], par, abort);
                    if (*abort) break;
                    mbar_arrive_expect_tx(&bar.v_full[st], S::TB);
                    copy(&bar.v_full[st], sv + st * S::TB, src + S::TB, S::TB);
                    ++values;
                }
            }
            // The last copies into each buffer have landed before the CTA ends: the issuing thread waits for them too, but may
            // have left after an error that this thread never saw. (Those before them were waited for with k_empty and v_empty.)
            for (int i = max(keys - 2, 0); i < keys; ++i) mbar_wait(&bar.k_full[i & 1], (i >> 1) & 1);
            for (int i = max(values - 2, 0); i < values; ++i) mbar_wait(&bar.v_full[i & 1], (i >> 1) & 1);
        }
        __syncwarp();
    } else if (!DENSE && warp == 1) {
        // ------------------------------ pages: a step's table entries, up to four steps ahead ------------------------------
        const Places at = places();
        PfBars& bar = at.bar;
        volatile int* const abort = at.abort;
        constexpr int RUNS = KT / 8;
        int it = 0;
        while (walk.next(a)) {
            if (__any_sync(0xffffffffu, *abort)) break;  // (all lanes: they meet at each step's ballot)
            const int row0 = walk.tile * R, rows = min(R, walk.fresh * a.G - row0);
            const int key_end = min(walk.base + (row0 + rows - 1) / a.G + 1, room);
            const int seen_from = a.window ? max(walk.base + row0 / a.G + 1 - a.window, 0) : 0;
            for (int t = walk.st0; t < walk.st1; ++t, ++it) {
                const int slot = it & 3, key0 = (walk.lo + t) * KT, key = key0 + (lane % RUNS) * 8;
                uint32_t row = KV4_NONE;
                bool gone = false;
                if (key < key_end && key + 8 > seen_from) {  // (what lies behind a window may have been freed)
                    const int pg = key / a.pool.page, id = a.table[(size_t)walk.b * a.width + pg];
                    gone = unsigned(id) >= unsigned(a.pool.pages);
                    if (gone)
                        record_status(LQ_DEV_BOUNDS);
                    else
                        row = kv4_row(a.pool, id, walk.kvh, key - pg * a.pool.page);
                }
                const uint32_t all_gone = __ballot_sync(0xffffffffu, lane < RUNS && gone);
                pf_wait(&bar.r_empty[slot], ((it >> 2) & 1) ^ 1, abort);
                if (lane < RUNS) bar.run[slot][lane] = row;
                if (lane == 0) {
                    bar.left[slot] = max(key_end - key0, 1);  // (a step that sees no key has no runs either)
                    bar.gone[slot] = all_gone;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.r_full[slot]);
            }
        }
        pf_wait(&bar.r_empty[it & 3], ((it >> 2) & 1) ^ 1, abort);
        if (lane == 0) {
            bar.left[it & 3] = 0;  // no more
            mbar_arrive(&bar.r_full[it & 3]);
        }
        __syncwarp();
    } else if (tid == 0) {
        // ------------------------------ MMA issuer: one thread ------------------------------
        const Places at = places();
        PfBars& bar = at.bar;
        volatile int* const abort = at.abort;
        const uint32_t tmem = at.tmem, sq = at.sq, sk = at.sk, sv = at.sv;
        constexpr uint32_t id_s = umma_idesc_f16(0, 128, KT);
        constexpr uint32_t id_o = umma_idesc_f16(0, 128, D) | (1u << 16);  // B's N side contiguous
        int it = 0, used[2] = {0, 0}, items[2] = {0, 0};
        // (descriptors: a start address in 16-byte units in the low word, the rest the same for all)
        const uint32_t d_q = uint32_t(umma_desc_sw128(sq)), d_k = uint32_t(umma_desc_sw128(sk));
        const uint32_t d_v = uint32_t(pf_desc_v(sv, S::SLAB));
        const uint32_t hi = uint32_t(umma_desc_sw128(0) >> 32);  // (both kinds')
        auto scores = [&](int w, int buf, int st) {
            pf_scores<D, S::SLAB>(tmem + buf * KT, d_q + w * (S::QB / 16), d_k + st * (S::TB / 16), hi, id_s,
                                  std::make_integer_sequence<int, D / 16>());
            tc_commit(&bar.s_full[buf]);
        };
        auto products = [&](int w, int buf, int st, bool first) {
            pf_products(tmem + S::O_COL + w * D, tmem + buf * KT, d_v + st * (S::TB / 16), hi, id_o, first ? 0u : 1u,
                        std::make_integer_sequence<int, KT / 16>());
            tc_commit(&bar.o_done[w]);
        };
        for (;;) {
            pf_wait(&bar.q_full[0], items[0]++ & 1, abort);
            const int rows = *reinterpret_cast<volatile int*>(&bar.rows), steps = *reinterpret_cast<volatile int*>(&bar.steps);
            if (rows == 0 || *abort) break;
            const int nq = rows > 128 ? 2 : 1;
            if (nq == 2) pf_wait(&bar.q_full[1], items[1]++ & 1, abort);
            if constexpr (NQ == 2) {
                pf_wait(&bar.k_full[it & 1], (it >> 1) & 1, abort);
                tc_fence_after();
                for (int w = 0; w < nq; ++w) scores(w, w, it & 1);
                tc_commit(&bar.k_empty[it & 1]);
                for (int t = 0; t < steps; ++t, ++it) {
                    const int st = it & 1, nx = (it + 1) & 1;
                    pf_wait(&bar.v_full[st], (it >> 1) & 1, abort);
                    for (int w = 0; w < nq; ++w) {
                        pf_wait(&bar.p_full[w], used[w]++ & 1, abort);
                        tc_fence_after();
                        products(w, w, st, t == 0);
                        if (t + 1 < steps) {
                            if (w == 0) {
                                pf_wait(&bar.k_full[nx], ((it + 1) >> 1) & 1, abort);
                                tc_fence_after();
                            }
                            scores(w, w, nx);
                        }
                    }
                    tc_commit(&bar.v_empty[st]);
                    if (t + 1 < steps) tc_commit(&bar.k_empty[nx]);
                }
            } else {
                for (int t = 0; t <= steps; ++t) {
                    if (t < steps) {
                        const int i = it + t;
                        pf_wait(&bar.k_full[i & 1], (i >> 1) & 1, abort);
                        tc_fence_after();
                        scores(0, (used[0] + t) & 1, i & 1);
                        tc_commit(&bar.k_empty[i & 1]);
                    }
                    if (t > 0) {
                        const int i = it + t - 1, u = used[0] + t - 1;
                        pf_wait(&bar.v_full[i & 1], (i >> 1) & 1, abort);
                        pf_wait(&bar.p_full[u & 1], (u >> 1) & 1, abort);
                        tc_fence_after();
                        products(0, u & 1, i & 1, t == 1);
                        tc_commit(&bar.v_empty[i & 1]);
                    }
                }
                it += steps;
                used[0] += steps;
            }
        }
        grid_dep_launch();
        tc_commit(&bar.done);  // nothing of this CTA's is in flight when its tensor memory goes (after an error too)
        mbar_wait(&bar.done, 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(*reinterpret_cast<volatile uint32_t*>(&tmem_base), 512);
    }
}

// One warp a (share, row): the parts of the item that a share's start divides, joined with the row's sink.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_prefill_join_kernel(const Kv4AttArgs a) {
    grid_dep_wait();
    const int i = blockIdx.x, j = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int32_t* rec = a.records + i * 8;
    if (!rec[0] || j >= rec[3]) return;
    const int row = rec[2] + j, qi = row / a.G, head = rec[4] * a.G + row - qi * a.G;
    kv4_join_row<T, D, 1>(a, PfShape<D>::R, j, i - 1, rec[5], 0, kv4_sink(a.sinks, head),
                          a.out + ((size_t)(rec[1] + qi) * a.H + head) * D, nullptr, nullptr);
}

// ---- host ----------------------------------------------------------------------------------------

// Unpack first where a request can have more than two tiles of rows, so that its keys would be unpacked again for each, and
// all keys that the table can name fit 1 GiB as fp16 tiles. 4,096 new tokens (128 tiles): 1,218 us in place, 1,057 unpacked
// first. 4 requests of 8,192 keys, 4 kv heads, D = 128, in place and first: one tile 61 and 80 us, two 88 and 101, three 117
// and 120, four 163 and 153.
static bool pf_dense(int D, int B, int KVH, int G, int max_q, long long room, size_t* bytes, int* steps) {
    const int R = D == 256 ? 128 : 256, KT = D == 256 ? 64 : 128;
    const long long n = (room + KT - 1) / KT, tiles = n * B * KVH;
    *steps = int(n);
    *bytes = size_t(tiles) * (size_t(4) * KT * D + 2 * KT + sizeof(int2));
    return (long long)max_q * G > 2 * R && tiles <= (1LL << 30) / (4LL * KT * D) && B <= 65535 && KVH <= 65535;
}

bool kv4_prefill_dense(int D, int B, int KVH, int G, int max_q, long long room) {
    size_t bytes;
    int steps;
    return pf_dense(D, B, KVH, G, max_q, room, &bytes, &steps);
}

static size_t pf_parts_bytes(int D, int sms) {
    const int R = D == 256 ? 128 : 256;
    return (size_t(sms) * 2 * R * (2 + D) * sizeof(float) + size_t(sms) * 8 * sizeof(int32_t) + 127) / 128 * 128;
}

size_t kv4_prefill_workspace_bytes(int D, int sms, int B, int KVH, int G, int max_q, long long room) {
    size_t bytes;
    int steps;
    return pf_parts_bytes(D, sms) + (pf_dense(D, B, KVH, G, max_q, room, &bytes, &steps) ? (bytes + 127) / 128 * 128 : 0);
}

template <typename T, int D>
static int kv4_prefill_d(Kv4AttArgs a, void* workspace, cudaStream_t st) {
    using S = PfShape<D>;
    static std::atomic<uint32_t> set{0}, set_dense{0}, set_first{0}, none{0};
    const int n = device_info().sm_count;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + size_t(n) * 2 * S::R * D;
    a.records = reinterpret_cast<int32_t*>(a.part_ml + size_t(n) * 2 * S::R * 2);
    size_t bytes;
    const size_t smem = S::SMEM + sizeof(PfBars);
    // One CTA a SM, but within 196 KB with the static arrays and what the system keeps: beyond, the rest of the SM's 256 KB
    // that is left to the L1 falls from 60 KB to 28, less than the stacks (a 4096-token prompt piece 1137 -> 1290 us).
    static_assert(S::SMEM + sizeof(PfBars) + 2 * 1024 <= 196 * 1024, "shared memory");
    int rc;
    if (pf_dense(D, a.B, a.pool.KVH, a.G, a.max_q, (long long)a.width * a.pool.page, &bytes, &a.dense_steps)) {
        a.dense = static_cast<uint8_t*>(workspace) + pf_parts_bytes(D, n);
        const size_t tiles = size_t(a.dense_steps) * a.B * a.pool.KVH;
        a.dense_keys = reinterpret_cast<int8_t*>(a.dense + tiles * 2 * S::TB);
        a.dense_meta = reinterpret_cast<int2*>(a.dense_keys + tiles * 2 * S::KT);
        rc = kv4_launch(kv4_dense_kernel<T, D>, set_first, dim3(a.dense_steps, a.pool.KVH, a.B), dim3(PD_WARPS * 32),
                        2 * S::TB + 128, st, a);
        if (!rc) rc = kv4_launch(kv4_prefill_kernel<T, D, true>, set_dense, dim3(n), dim3(pf_threads(true)), smem, st, a);
    } else {
        rc = kv4_launch(kv4_prefill_kernel<T, D, false>, set, dim3(n), dim3(pf_threads(false)), smem, st, a);
    }
    if (rc) return rc;
    return kv4_launch(kv4_prefill_join_kernel<T, D>, none, dim3(n, S::R / 4), dim3(128), 0, st, a);
}

int kv4_prefill_run(const Kv4AttArgs& a, int D, int dtype, void* workspace, cudaStream_t st) {
    if (dtype == LQ_BF16)
        return D == 64    ? kv4_prefill_d<__nv_bfloat16, 64>(a, workspace, st)
               : D == 128 ? kv4_prefill_d<__nv_bfloat16, 128>(a, workspace, st)
                          : kv4_prefill_d<__nv_bfloat16, 256>(a, workspace, st);
    return D == 64    ? kv4_prefill_d<__half, 64>(a, workspace, st)
           : D == 128 ? kv4_prefill_d<__half, 128>(a, workspace, st)
                      : kv4_prefill_d<__half, 256>(a, workspace, st);
}

}  // namespace lq
