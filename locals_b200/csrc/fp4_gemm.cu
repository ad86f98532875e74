// Products with microscaled 4-bit weights on the block-scaled tensor cores of sm_100a: y (M, N) = x . w^T, x in the same
// 4-bit format, or in 16 bits (experts' hidden rows: 32) against mxfp4 weights; dense, or grouped over the experts that rows are
// routed to.
//
// Mathematics. Each value of a group is code * scale, so a group's part of a sum is scale_x scale_w sum code_x code_w, and
// the tensor core does all of it: the products of codes are exact, the scales enter as operands, sums are 32 bits. No
// weight is ever unpacked. Activations of 16 bits are first split in pieces of e4m3 (4 significant bits), each with a power
// of two a group of 32: bf16 (8 bits) is the sum of 2, fp16 (11 bits) of 3. With E the exponent of the largest magnitude of
// the group, piece p has the scale 2^(E - 7 - 5 p) (its values are below 2^8, so what is left after rounding them to 4 bits
// is at most 2^3) and is the rounded remainder of those before it. The pieces' sum is x exactly down to 2^-14 of that
// magnitude; below, it is off by about half a last step, less than 2^-21 (bf16) or 2^-26 (fp16) of it, less than
// the 32-bit sum itself loses beside that value. A group that holds an infinity or no number is not a number. Values of 32 bits
// (the hidden rows between experts' two products, which lq_fp4_moe does not round) enter as three pieces: off by at most 2^-14 of
// themselves, 1/32 of a rounding to bf16 and 1/4 of one to fp16. Two pieces would do for bf16 but for 7% more error in all.
//
// Layout. Weights are the MMA's A operand (128 rows of w a tile, one a tensor-memory lane), T tokens its N side, so that one
// token costs a narrow MMA and not a row of an empty tile. Warp 8 streams a ring of stages by TMA, 128 bytes of every row (256
// codes; against e4m3, 128 codes that TMA spreads to bytes), warp 10 their scale tiles. Warp 9 copies the scales to tensor
// memory and issues the MMAs; warps 0 to 7 write finished tiles out under the next tile's MMAs. The scales have two places in
// tensor memory: a stage's are copied only when the MMAs of the stage before last are done. (Copies from a warp of their
// own queue behind the other warp's MMAs: 2,048 tokens by 14336 x 4096 172 -> 196 us.)
// Few tiles: a cluster of CTAs splits a tile's K and joins its sums through distributed shared memory, in rank order.
// Many tokens: a pair of CTAs has 256 rows of w by 256 (128) tokens, each CTA half of either, so that an operand's byte is
// read from L2 half as often. Two accumulators of 256 columns share 128, since scales take the rest of tensor memory.
//
// Measured on a B200 (captured graphs; floors at 6,458 GB/s and 1,653 TFLOP/s of bf16, four times that for 4 by 4 bits):
// both in nvfp4, 4,096 tokens by 14336 x 4096 111 to 113 us (4.3 PFLOP/s; 130 over 1.6 s, the SMs at 1,597 MHz under the power
// limit), bound by the one thread that issues (12 scale copies and 4 MMAs a stage take it about as long as the MMAs run) and by
// the waits of a stage; the tensor pipe is busy 37 to 45% of the time. bf16 by mxfp4, 2,048 tokens by the same 170 us (1.4 PFLOP/s,
// 85% of the bf16 rate; 202 over 2.4 s at 1,537 MHz): the tensor pipe, 69% busy, and 7 rounds of tiles of which the last is 5% full;
// fp16, with three pieces, 249 us. One token by 14336 x 4096 9.3 us and by 6144 x 2560 5.9 us, weights rotated through more than
// L2 or not (9.3 and 5.8 over three sets): start, first loads and join, some 4 us whatever the size; one launch alone and cold
// takes the former 15.6 us (the profile).
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "fp4.cuh"
#include "fp4_host.h"
#include "lq_host.h"

namespace lq {

constexpr int FP4_OUT = 8;                           // warps that write tiles out
constexpr int FP4_THREADS = 32 * (FP4_OUT + 3);
constexpr int FP4_MAX_STAGES = 10;
constexpr int FP4_MAX_SEGMENTS = 1024;
constexpr int FP4_FUSE_SMS = 148;  // (fixed, so that a workspace's size does not need the device)

// A grouped call's segments in shared memory: n of them, their first rows and experts, and the tiles of tokens before each.
struct Fp4Segments {
    int n;
    int32_t starts[FP4_MAX_SEGMENTS + 1], tiles[FP4_MAX_SEGMENTS + 1], experts[FP4_MAX_SEGMENTS];
};

// X_: the type of x where the product makes its pieces itself, else void.
template <int KIND_, int P_, int T_, int CG_ = 1, typename X_ = void>
struct Fp4Shape {
    using X = X_;
    static constexpr int KIND = KIND_, P = P_, T = T_;
    static constexpr int CG = CG_;  // CTAs a tile: a pair has 128 rows of w and half of the tokens each
    static constexpr bool STACK = KIND == FP4_SPLIT && T <= 32;  // a token's pieces are columns of one MMA
    // Few tokens of 16 bits and no more tiles than run at once: four warps make the pieces in shared memory, with no kernel before
    // this one (one token and 6144 x 2560: 9.2 -> 6.6 us). With more tiles each CTA makes the same pieces again (64 tokens
    // over 64 experts: 57 us with a kernel that makes them once, 65 without).
    static constexpr bool FUSE = !std::is_same<X, void>::value;
    static constexpr int OUT = FUSE ? 4 : FP4_OUT;  // warps that write out
    static constexpr int TURN = KIND == FP4_SPLIT ? 1024 : 2048;  // bytes of a warp for tokens on their way: 16 (of 32 bits 8 or 16)
    static constexpr int BK = KIND == FP4_SPLIT ? 128 : 256;     // values a stage
    static constexpr int KB = KIND == FP4_MX ? 2 : KIND == FP4_NV ? 4 : 1;  // scale tiles a stage and 128 rows
    static constexpr int NB = STACK ? 1 : P * ((T + 127) / 128);            // scale tiles of x beside each of w's
    static constexpr int A_BYTES = 128 * 128, B_TILE = T / CG * 128, B_BYTES = P * B_TILE;
    // what TMA counts of a weight tile: the bytes that it reads, also where it spreads codes to bytes
    static constexpr int A_TX = KIND == FP4_SPLIT ? A_BYTES / 2 : A_BYTES;
    static constexpr int SFA = KB * 512, SFB = KB * NB * 512;
    static constexpr int TX = A_TX + SFA + (FUSE ? 0 : B_BYTES + SFB);  // bytes that arrive for a stage (in each CTA)
    static constexpr int STAGE = (A_BYTES + B_BYTES + SFA + SFB + 1023) / 1024 * 1024;
    // shared memory beside the ring (segs: of a grouped call), and the ring's stages in what is left: of the SM's 227 KB, or
    // of a half where tiles are narrow and two CTAs share it
    static constexpr size_t beside(bool segs) { return 1024 + (2 * FP4_MAX_STAGES + 4) * 8 + 32 + OUT * TURN + (segs ? sizeof(Fp4Segments) : 0); }
    static constexpr int stages(bool segs) {
        const int n = int(((T <= 32 ? 113 : 227) * 1024 - beside(segs)) / STAGE);
        return n < FP4_MAX_STAGES ? n : FP4_MAX_STAGES;
    }
    static constexpr int N = STACK ? P * T : T;
    static constexpr int ACC = N <= 32 ? 32 : N <= 64 ? 64 : N <= 96 ? 96 : N <= 128 ? 128 : 256;
    // 256 columns: the two accumulators share 128, which are read out first
    static constexpr int ACC_STEP = ACC == 256 ? 128 : ACC;
    static constexpr int SF_COL = ACC == 256 ? 384 : 2 * ACC, SF_COLS = 4 * KB * (1 + NB);
    static constexpr int COLS = SF_COL + 2 * SF_COLS, TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static_assert(COLS <= 512 && stages(true) >= 2 && N % 16 == 0 && N <= 256 && B_TILE % 1024 == 0, "tile");
    static_assert(!FUSE || STACK, "few tokens");
    // Two CTAs of an SM both have their tensor memory, so that neither waits for the other's work.
    static_assert(T > 32 || TMEM <= 256, "two CTAs an SM");
    static_assert(!STACK || N <= 128, "stacked pieces share one scale tile");
};

struct Fp4Args {
    int M, N, Kp;        // rows of x, rows of w (of an expert), padded K
    int ns, ktiles;      // stages along K, scale tiles along K
    int ntn, ntiles;     // tiles along N, all tiles (dense)
    int rtiles;          // scale tiles along N
    int ks;              // CTAs that split a tile's K
    int nst;             // stages of the ring
    int glu, dtype;
    int piece_rows;      // rows of one piece of x
    const float* xf;     // factors, or NULL
    const float* wf;
    void* y;
    // x before it is split (few tokens)
    const void* x_rows;
    int64_t x_row;
    int K, vec, gather, src_rows;  // vec: rows start on 16-byte boundaries
    const int32_t* order;          // gather > 0: row j is row order[j] / gather of x (order NULL: j / gather); 0: row j
    // grouped
    int grouped, E;
    const int32_t* starts;
    const int32_t* experts;
    const int32_t* nseg;
    int max_seg;
};

// A tile's rows [r0, r1) of x.
struct Fp4Tile {
    int n0, r0, r1;   // first row of w (of the expert), rows of x
    int expert, id;   // id: the tile of x's scales (segment s has starts[s] / T + s, ...; a number may go unused)
};

template <typename S>
__device__ __forceinline__ bool fp4_tile(const Fp4Args& a, const Fp4Segments& seg, int lin, Fp4Tile& t) {
    constexpr int T = S::T, ROWS = 128 * S::CG;
    if (!a.grouped) {
        const int mt = a.ntiles / a.ntn;
        t.id = lin % mt;  // token tiles next to one another in time share the weights
        t.n0 = lin / mt * ROWS;
        t.r0 = t.id * T;
        t.r1 = min(a.M, t.r0 + T);
        t.expert = 0;
        return true;
    }
    const int q = int(uint32_t(lin) / uint32_t(a.ntn));
    t.n0 = (lin - q * a.ntn) * ROWS;
    int lo = 0, hi = seg.n;  // the last segment whose first tile is not beyond q
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (seg.tiles[mid] <= q) lo = mid; else hi = mid;
    }
    const int first = seg.starts[lo], i = q - seg.tiles[lo];
    t.id = int(uint32_t(first) / T) + lo + i;
    t.r0 = first + i * T;
    t.r1 = min(seg.starts[lo + 1], t.r0 + T);
    t.expert = seg.experts[lo];
    if (t.expert == a.E) return false;  // padding
    if (t.expert < 0 || t.expert > a.E) {
        record_status(LQ_DEV_BOUNDS);
        return false;
    }
    return true;
}

// x / (1 + e^-x), below 0 as x e^x / (1 + e^x), so that no exponential overflows and the divisor is 1 to 2: some four units in the
// last place, down to where e^x is no normal number (-87.3; its own step there, 2^-149, times x). (The fast exponential's error
// grows with |x|: 25 units at -20, some 95 at -80.)
__device__ __forceinline__ float fp4_silu(float x) {
    const float t = expf(-fabsf(x)), s = __fdividef(x, 1.f + t);
    return x < 0.f ? s * t : s;
}

// The product of the matrices' factors, as two numbers to multiply a sum by in turn: the second is 1 but where the product is
// beyond 2^120 or below 2^-121. Multiplied first, factors of 1e-22 each were 0 or a few bits, and two of 1e25 an infinity,
// whatever the sum is.
__device__ __forceinline__ float2 fp4_factors(const Fp4Args& a) {
    int ex, ew;
    const float mx = frexpf(a.xf ? *a.xf : 1.f, &ex), mw = frexpf(a.wf ? *a.wf : 1.f, &ew);
    const float m = mx * mw;
    if (!(fabsf(m) < 1.f)) return make_float2(m, 1.f);  // (an infinity or no number)
    const int e = ex + ew, e1 = max(-120, min(120, e));
    return make_float2(ldexpf(m, e1), ldexpf(1.f, max(-126, min(126, e - e1))));
}

__device__ __forceinline__ void fp4_store(const Fp4Args& a, int64_t at, float v) {
    if (a.dtype == LQ_F32)
        reinterpret_cast<float*>(a.y)[at] = v;
    else if (a.dtype == LQ_BF16)
        reinterpret_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
    else
        reinterpret_cast<__half*>(a.y)[at] = __float2half_rn(v);
}

// Output column c of a tile: row n of w, v its sum. glu: rows of w are gate 0, up 0, gate 1, ...: neighbouring lanes.
template <typename S>
__device__ __forceinline__ void fp4_out(const Fp4Args& a, const Fp4Tile& t, int c, int n, float v) {
    if (a.glu) {
        const float up = __shfl_xor_sync(0xFFFFFFFFu, v, 1);
        if (!(n & 1) && n < a.N && t.r0 + c < t.r1) fp4_store(a, int64_t(t.r0 + c) * (a.N / 2) + n / 2, fp4_silu(v) * up);
    } else if (n < a.N && t.r0 + c < t.r1) {
        fp4_store(a, int64_t(t.r0 + c) * a.N + n, v);
    }
}

// 16 output columns (tokens) of a warp's 32 rows of w, v[c] the value of this lane's row and token c0 + c: turned to rows of y
// through shared memory, so that a token's 32 values leave in pieces of 16 bytes. Neighbouring lanes first swap
// columns: the even lane then has two rows of an even column, the odd lane two of an odd one. The type and form are fixed
// here, not asked for at each value: with branches between the shuffles they ran one after another (1,670 cycles, not 150).
template <typename O, bool GLU, int TURN>
__device__ __forceinline__ void fp4_out16_t(const Fp4Args& a, const Fp4Tile& t, int c0, int nb, const float (&v)[16], uint8_t* stage,
                                            int lane) {
    constexpr int BYTES = (GLU ? 16 : 32) * int(sizeof(O)), PER = BYTES / 16;  // of a token's values here
    const bool odd = lane & 1;
    const int64_t width = GLU ? a.N / 2 : a.N;
    O* y = static_cast<O*>(a.y) + int64_t(t.r0 + c0) * width + (GLU ? nb / 2 : nb);
    const int rows = t.r1 - t.r0 - c0;
    auto leave = [&](int c_lo, auto count) {  // `count` tokens from c_lo on
        constexpr int PIECES = decltype(count)::value * PER;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < (PIECES + 31) / 32; ++i) {
            const int q = lane + 32 * i, c = c_lo + q / PER;
            if (c < rows && q < PIECES)
                *reinterpret_cast<uint4*>(y + c * width + (q % PER) * (16 / int(sizeof(O)))) = *reinterpret_cast<uint4*>(stage + q * 16);
        }
        __syncwarp();
    };
    if constexpr (sizeof(O) == 4 && !GLU) {
        constexpr int AT = TURN / BYTES < 16 ? TURN / BYTES : 16;  // tokens that fit
#pragma unroll
        for (int c1 = 0; c1 < 16; c1 += AT) {
#pragma unroll
            for (int c = 0; c < AT; ++c) reinterpret_cast<float*>(stage + c * BYTES)[lane] = v[c1 + c];
            leave(c1, std::integral_constant<int, AT>());
        }
    } else {
        static_assert(16 * BYTES <= TURN, "16 tokens fit");
        float got[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) got[c] = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2 * c] : v[2 * c + 1], 1);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float mine = odd ? v[2 * c + 1] : v[2 * c], lo = odd ? got[c] : mine, hi = odd ? mine : got[c];
            uint8_t* row = stage + (2 * c + odd) * BYTES;
            if constexpr (GLU) {
                const float h = fp4_silu(lo) * hi;
                if constexpr (sizeof(O) == 4)
                    reinterpret_cast<float*>(row)[lane >> 1] = h;
                else
                    reinterpret_cast<uint16_t*>(row)[lane >> 1] = F16Traits<O>::from_f32(h);
            } else {
                reinterpret_cast<uint32_t*>(row)[lane >> 1] = F16Traits<O>::pack2(hi, lo);
            }
        }
        leave(0, std::integral_constant<int, 16>());
    }
}

template <int TURN>
__device__ __forceinline__ void fp4_out16(const Fp4Args& a, const Fp4Tile& t, int c0, int nb, const float (&v)[16], uint8_t* stage,
                                          int lane) {
    if (a.glu) {
        if (a.dtype == LQ_BF16)
            fp4_out16_t<__nv_bfloat16, true, TURN>(a, t, c0, nb, v, stage, lane);
        else if (a.dtype == LQ_F16)
            fp4_out16_t<__half, true, TURN>(a, t, c0, nb, v, stage, lane);
        else
            fp4_out16_t<float, true, TURN>(a, t, c0, nb, v, stage, lane);
    } else {
        if (a.dtype == LQ_BF16)
            fp4_out16_t<__nv_bfloat16, false, TURN>(a, t, c0, nb, v, stage, lane);
        else if (a.dtype == LQ_F16)
            fp4_out16_t<__half, false, TURN>(a, t, c0, nb, v, stage, lane);
        else
            fp4_out16_t<float, false, TURN>(a, t, c0, nb, v, stage, lane);
    }
}

// Four neighbouring rows of w (two pairs of gate and up) and one token.
__device__ __forceinline__ void fp4_out4(const Fp4Args& a, const Fp4Tile& t, int c, int n, float4 v) {
    float o[4] = {v.x, v.y, v.z, v.w};
    const int width = a.glu ? a.N / 2 : a.N, at = a.glu ? n / 2 : n, some = a.glu ? 2 : 4;
    if (a.glu) {
        o[0] = fp4_silu(o[0]) * o[1];
        o[1] = fp4_silu(o[2]) * o[3];
    }
    const int64_t first = int64_t(t.r0 + c) * width + at;
    if (a.dtype != LQ_F32 && !a.glu && width % 4 == 0 && n + 4 <= a.N && reinterpret_cast<uintptr_t>(a.y) % 8 == 0) {
        uint2 w = a.dtype == LQ_BF16 ? make_uint2(cvt_bf16x2(o[1], o[0]), cvt_bf16x2(o[3], o[2]))
                                     : make_uint2(cvt_f16x2(o[1], o[0]), cvt_f16x2(o[3], o[2]));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + first) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < some && at + i < width) fp4_store(a, first + i, o[i]);
}

// 8 values of a group of 32 (four lanes next to one another) to P pieces of e4m3 bytes and their scale bytes. Scaled to below
// 2^8, 16-bit values are fp16 numbers but for what lies below 2^-24 there, and the steps from piece to piece are exact in fp16;
// 32-bit values take theirs in 32 bits.
template <typename X, int P>
__device__ __forceinline__ void split8(const Eight<X>& x, uint32_t mask, uint2 (&piece)[P], int (&byte)[P]) {
    float top = x.amax();
#pragma unroll
    for (int d = 1; d < 4; d *= 2) top = amax_nan(top, __shfl_xor_sync(mask, top, d));
    const uint32_t e = __float_as_uint(top) >> 23 & 0xFF;
    byte[0] = e == 255 ? 255 : e < 7 ? 0 : int(e) - 7;
    const float up = __uint_as_float((254u - (e == 255 ? 127u : uint32_t(byte[0]))) << 23);
    float v[8];
    x.times(up, v);
    __half2 h[4];
    if constexpr (sizeof(X) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        uint16_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(X) == 2)
                asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(q[i]) : "r"(*reinterpret_cast<uint32_t*>(&h[i])));
            else
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(q[i]) : "f"(v[2 * i]), "f"(v[2 * i + 1]));
        }
        asm("mov.b32 %0, {%1, %2};" : "=r"(piece[p].x) : "h"(q[0]), "h"(q[1]));
        asm("mov.b32 %0, {%1, %2};" : "=r"(piece[p].y) : "h"(q[2]), "h"(q[3]));
        if (p + 1 < P) {
            byte[p + 1] = byte[p] == 255 ? 255 : byte[p] < 5 ? 0 : byte[p] - 5;
            const float more = __uint_as_float(uint32_t(127 + (byte[p] == 255 ? 0 : byte[p] - byte[p + 1])) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(X) == 2) {
                    uint32_t back;
                    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(q[i]));
                    h[i] = __hmul2(__hsub2(h[i], *reinterpret_cast<__half2*>(&back)), __float2half2_rn(more));
                } else {
                    const float2 back = e4m3x2_to_f32(q[i]);
                    v[2 * i] = (v[2 * i] - back.x) * more;
                    v[2 * i + 1] = (v[2 * i + 1] - back.y) * more;
                }
            }
        }
    }
}

// The tensor maps of a product: codes of w and x (or pieces of x), scale tiles of w and x.
struct Fp4Maps {
    CUtensorMap w, x, ws, xs;
};

template <typename S>
__global__ void __launch_bounds__(FP4_THREADS, S::T <= 32 ? 2 : 1) fp4_gemm_kernel(const __grid_constant__ Fp4Maps m, const Fp4Args a) {
    constexpr int T = S::T, P = S::P, CG = S::CG;
    const int NS = a.nst;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + NS * S::STAGE);  // (in a pair, the lower rank's, for both)
    uint64_t* empty = full + NS;
    uint64_t* acc_full = empty + NS;     // [2] the MMAs of a tile are done
    uint64_t* acc_empty = acc_full + 2;  // [2] the epilogue has read what the next tile writes
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    uint8_t* stage = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tmem_slot + 1) + 15) & ~uintptr_t(15));
    Fp4Segments& seg = *reinterpret_cast<Fp4Segments*>(stage + S::OUT * S::TURN);  // (grouped)

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = CG == 2 || a.ks > 1 ? int(cluster_ctarank()) : 0;
    const int share = CG == 2 ? 2 : a.ks, half = CG == 2 ? rank : 0;
    const int first = int(blockIdx.x) / share, step = int(gridDim.x) / share;
    const int s_lo = CG == 2 ? 0 : a.ns * rank / a.ks, s_hi = CG == 2 ? a.ns : a.ns * (rank + 1) / a.ks;  // stages of a tile

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], S::FUSE ? 2 : 1);
            mbar_init(&empty[s], 1);
        }
        for (int j = 0; j < 2; ++j) {
            mbar_init(&acc_full[j], 1);
            mbar_init(&acc_empty[j], S::OUT * CG);
        }
        fence_barrier_init();
    }
    if (warp == FP4_OUT + 1) tc_alloc<CG>(tmem_slot, S::TMEM);
    if (a.grouped) {
        grid_dep_wait();
        const int n = a.nseg ? min(max(*a.nseg, 0), a.max_seg) : a.M;  // without segments, each row is one
        for (int i = threadIdx.x; i <= n; i += FP4_THREADS) seg.starts[i] = a.starts ? min(max(a.starts[i], 0), a.M) : i;
        for (int i = threadIdx.x; i < n; i += FP4_THREADS) seg.experts[i] = a.experts[i];
        if (threadIdx.x == 0) {
            seg.n = n;
            if (a.nseg && *a.nseg != n) record_status(LQ_DEV_BOUNDS);  // a grouping of more experts than there are
        }
        __syncthreads();
        if (warp == 0) {  // tiles before each segment
            int before = 0;
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int i = i0 + lane;
                int v = i < n ? (max(seg.starts[i + 1] - seg.starts[i], 0) + T - 1) / T : 0, sum = v;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int o = __shfl_up_sync(0xFFFFFFFFu, sum, d);
                    if (lane >= d) sum += o;
                }
                if (i < n) seg.tiles[i] = before + sum - v;
                before += __shfl_sync(0xFFFFFFFFu, sum, 31);
            }
            if (lane == 0) seg.tiles[n] = before;
        }
    }
    tc_fence_before();
    // The cluster barrier counts warps: the one whose first lane sets up the mbarriers arrives when that lane has, not before
    // (a load ahead of the wait below met a barrier that was then set up again).
    __syncwarp();
    if constexpr (CG == 2)
        cluster_sync();
    else
        __syncthreads();
    tc_fence_after();
    grid_dep_launch();  // this CTA has its tensor memory: the next kernel's may wait for theirs
    const uint32_t tmem = *tmem_slot;
    const int ntiles = a.grouped ? seg.tiles[seg.n] * a.ntn : a.ntiles;
    bool ok = true;

    if (warp == FP4_OUT || warp == FP4_OUT + 2) {
        // ------------------------------ producers: codes (and pieces), and scales ------------------------------
        const bool scales = warp == FP4_OUT + 2;
        if (elect_one()) {
            prefetch_tmap(scales ? &m.ws : &m.w);
            if constexpr (!S::FUSE) prefetch_tmap(scales ? &m.xs : &m.x);
            const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
            const uint32_t ring = smem_u32(smem), bars = CG == 2 ? map_peer(smem_u32(full), 0) : smem_u32(full);
            int it = 0, s = 0, turn = 0;  // stages so far, the ring's next slot, rounds of the ring
            bool waited = a.grouped;
            Fp4Tile t;
            // one thread says what arrives for a stage in both CTAs; a copy may arrive before that
            auto expect = [&](int slot) {
                if (!scales && (CG == 1 || rank == 0)) mbar_arrive_expect_tx(&full[slot], CG * S::TX);
            };
            for (int lin = first; lin < ntiles && ok; lin += step) {
                if (!fp4_tile<S>(a, seg, lin, t)) continue;
                const int wrow = t.expert * a.N + t.n0 + 128 * half, wtile = t.expert * a.rtiles + t.n0 / 128 + half;
                auto weights = [&](int kb, int slot) {
                    const uint32_t st = ring + slot * S::STAGE, bar = bars + slot * 8;
                    if (!scales)
                        load_2d<CG>(st, &m.w, bar, kb * 128, wrow, pol_w);
                    else
                        load_3d<CG>(st + S::A_BYTES + S::B_BYTES, &m.ws, bar, 0, kb * S::KB, wtile, pol_w);
                };
                // Before this kernel came the split, which was launched on when the kernels before it were done: what they
                // wrote, weights too, may be read before the split ends. Without one, this may follow the kernel that
                // quantized the weights.
                int ahead = 0;
                if (!waited) {
                    for (; S::KIND == FP4_SPLIT && !S::FUSE && ahead < NS && s_lo + ahead < s_hi; ++ahead) {
                        expect(ahead);
                        weights(s_lo + ahead, ahead);
                    }
                    grid_dep_wait();
                    waited = true;
                }
                for (int kb = s_lo; kb < s_hi; ++kb, ++it, ++s) {
                    if (s == NS) {
                        s = 0;
                        ++turn;
                    }
                    if (turn > 0 && !(ok = mbar_wait_cg<CG>(&empty[s], (turn - 1) & 1))) break;
                    if (it >= ahead) {
                        expect(s);
                        weights(kb, s);
                    }
                    const uint32_t st = ring + s * S::STAGE + S::A_BYTES, bar = bars + s * 8;
                    if constexpr (S::FUSE) {
                    } else if (!scales) {
#pragma unroll
                        for (int p = 0; p < P; ++p)
                            load_2d<CG>(st + p * S::B_TILE, &m.x, bar, kb * 128, p * a.piece_rows + t.r0 + half * (T / CG), pol_x);
                    } else if constexpr (S::KIND == FP4_SPLIT) {
                        load_3d<CG>(st + S::B_BYTES + S::SFA, &m.xs, bar, 0, 0, t.id * a.ktiles + kb, pol_x);
                    } else {
                        load_3d<CG>(st + S::B_BYTES + S::SFA, &m.xs, bar, 0, kb * S::KB, t.r0 / 128, pol_x);
                    }
                }
            }
            // after a wait that gave up: the copies in flight land before the CTA's shared memory is another's
            if (!ok && !scales && (CG == 1 || rank == 0))
                for (int q = it > NS ? it - NS : 0; q < it; ++q) mbar_wait(&full[q % NS], (q / NS) & 1);
        }
        __syncwarp();
    } else if (warp == FP4_OUT + 1) {
        // ------------------------------ MMA issuer (in a pair, the lower rank's) ------------------------------
        constexpr uint32_t idesc = fp4_idesc<S::KIND>(128 * CG, S::N);
        constexpr int PP = S::STACK ? 1 : P;  // MMAs a step along K
        const bool lead = elect_one();
        const uint32_t ring = smem_u32(smem);
        const uint64_t a_desc = umma_desc_sw128(ring), b_desc = umma_desc_sw128(ring + S::A_BYTES);
        const uint64_t fa_desc = umma_desc_scales(ring + S::A_BYTES + S::B_BYTES);
        const uint64_t fb_desc = umma_desc_scales(ring + S::A_BYTES + S::B_BYTES + S::SFA);
        int it = 0, j = 0, s = 0, turn = 0;
        Fp4Tile t;
        for (int lin = first; (CG == 1 || rank == 0) && lin < ntiles && ok; lin += step) {
            if (!fp4_tile<S>(a, seg, lin, t)) continue;
            if constexpr (S::ACC == 256) {
                if (j >= 1) ok = mbar_wait_cg<CG>(&acc_empty[0], (j - 1) & 1);
            } else {
                if (j >= 2) ok = mbar_wait_cg<CG>(&acc_empty[j & 1], ((j >> 1) - 1) & 1);
            }
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem + uint32_t((j & 1) * S::ACC_STEP);
            for (int kb = s_lo; kb < s_hi && ok; ++kb, ++it, ++s) {
                if (s == NS) {
                    s = 0;
                    ++turn;
                }
                // the scales' place: the MMAs of the stage before last are done
                if (it >= 2) ok = mbar_wait_cg<CG>(&empty[s >= 2 ? s - 2 : s - 2 + NS], (s >= 2 ? turn : turn - 1) & 1);
                if (ok) ok = mbar_wait_cg<CG>(&full[s], turn & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t at = uint64_t(s * (S::STAGE / 16));
                const uint32_t sfa = tmem + S::SF_COL + uint32_t(it & 1) * S::SF_COLS, sfb = sfa + 4 * S::KB;
                const int kt = min(S::KB, a.ktiles - kb * S::KB);  // scale tiles of this stage: fewer in a row's last
                auto issue = [&](int q) {                          // a scale tile's MMAs
                    constexpr int PER = 4 / S::KB;
                    tc_copy_scales<CG>(sfa + 4 * q, fa_desc + at + q * 32);
#pragma unroll
                    for (int b = 0; b < S::NB; ++b)
                        tc_copy_scales<CG>(sfb + 4 * (q * S::NB + b), fb_desc + at + (b * S::KB + q) * 32);
#pragma unroll
                    for (int k = q * PER; k < (q + 1) * PER; ++k) {
                        const uint32_t id = fp4_idesc_byte(S::KIND == FP4_MX ? 2 * (k % 2) : S::KIND == FP4_NV ? 0 : k);
#pragma unroll
                        for (int p = 0; p < PP; ++p)
                            tc_mma_fp4<S::KIND, CG>(acc, a_desc + at + k * 2, b_desc + at + p * (S::B_TILE / 16) + k * 2, idesc | id,
                                                    sfa + 4 * q, sfb + 4 * (q * S::NB + p * (S::NB / PP)),
                                                    (kb > s_lo || k > 0 || p > 0) ? 1u : 0u);
                    }
                };
                if (lead) {
                    if (kt == S::KB) {
#pragma unroll
                        for (int q = 0; q < S::KB; ++q) issue(q);
                    } else {
#pragma unroll
                        for (int q = 0; q < S::KB - 1; ++q)
                            if (q < kt) issue(q);
                    }
                    tc_commit_all<CG>(&empty[s]);
                }
                __syncwarp();
            }
            if (lead) tc_commit_all<CG>(&acc_full[j & 1]);
            __syncwarp();
            ++j;
        }
    } else if (warp >= S::OUT) {
        // ------------------------------ converters: x to pieces ------------------------------
        // The warps take stages in turn, so that the loads of four stages are on their way; a lane takes 8 values of a token.
        // No more warps than the ring has stages: one that is `turns` stages on has then seen, at its last stage, the place of
        // the stage two rounds back handed over, and the parity that it waits for is not the one of two rounds before.
        if constexpr (S::FUSE) {
            using X = typename S::X;
            constexpr int AHEAD = 8 / int(sizeof(X));  // values of 8 that a lane loads before it converts (32-bit ones: 2)
            grid_dep_wait();
            const int turns = NS < 4 ? NS : 4, mine = warp - S::OUT, chunk = lane & 15;
            int who = 0, s = 0, turn = 0;  // the warp of the next stage, its place, rounds of the ring
            Fp4Tile t;
            for (int lin = first; lin < ntiles && ok; lin += step) {
                if (!fp4_tile<S>(a, seg, lin, t)) continue;
                int src = t.r0 + lane < t.r1 ? t.r0 + lane : -1;  // the row of x of the tile's token `lane`
                if (a.gather && src >= 0) {
                    const int pair = a.order ? a.order[src] : src;
                    src = pair < 0 ? -1 : pair / a.gather;
                }
                if (src >= a.src_rows || (src < 0 && t.r0 + lane < t.r1)) {
                    record_status(LQ_DEV_BOUNDS);
                    src = -1;  // zeros
                }
                const int tasks = (t.r1 - t.r0 + 1) / 2;  // of two tokens
                for (int kb = s_lo; kb < s_hi; ++kb, ++who, ++s) {
                    if (s == NS) {
                        s = 0;
                        ++turn;
                    }
                    if (who == turns) who = 0;
                    if (who != mine) continue;
                    bool free = turn == 0;
                    uint8_t* b = smem + s * S::STAGE + S::A_BYTES;
                    for (int i0 = 0; i0 < tasks; i0 += AHEAD) {
                        Eight<X> v[AHEAD];
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) {
                            const int row = __shfl_sync(0xFFFFFFFFu, src, (2 * (i0 + i) + (lane >> 4)) & 31);
                            v[i].zero();
                            if (i0 + i < tasks && row >= 0)
                                v[i].load(static_cast<const X*>(a.x_rows) + int64_t(row) * a.x_row, kb * 128 + chunk * 8, a.K, a.vec);
                        }
                        if (!free && !(ok = mbar_wait(&empty[s], (turn - 1) & 1))) break;
                        free = true;
                        auto put = [&](int i, const uint2(&piece)[P], const int(&byte)[P]) {
#pragma unroll
                            for (int p = 0; p < P; ++p) {
                                const int r = p * T + 2 * i + (lane >> 4);  // 128-byte rows, their 16-byte pieces swizzled
                                *reinterpret_cast<uint2*>(b + r * 128 + (((chunk >> 1) ^ (r & 7)) << 4) + (chunk & 1) * 8) = piece[p];
                                if (chunk % 4 == 0) b[S::B_BYTES + S::SFA + fp4_tile_byte(r, chunk / 4)] = uint8_t(byte[p]);
                            }
                        };
                        // two at a time where there are two: one is a chain of conversions (some 550 cycles)
#pragma unroll
                        for (int i = 0; i < AHEAD; i += 2) {
                            uint2 p0[P], p1[P];
                            int b0[P], b1[P];
                            if (i0 + i + 1 < tasks) {
                                split8<X, P>(v[i], 0xFFFFFFFFu, p0, b0);
                                split8<X, P>(v[i + 1], 0xFFFFFFFFu, p1, b1);
                                put(i0 + i, p0, b0);
                                put(i0 + i + 1, p1, b1);
                            } else if (i0 + i < tasks) {
                                split8<X, P>(v[i], 0xFFFFFFFFu, p0, b0);
                                put(i0 + i, p0, b0);
                            }
                        }
                    }
                    if (!ok) break;
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[s]);
                }
            }
        }
    } else {
        // ------------------------------ epilogue: two warps (few 16-bit tokens: one) a quarter of the lanes ------------------------------
        grid_dep_wait();
        const float2 f = S::KIND == FP4_SPLIT ? make_float2(1.f, 1.f) : fp4_factors(a);
        // 16-byte pieces of y: its rows start on 16-byte boundaries
        const int ysize = (a.glu ? a.N / 2 : a.N) * (a.dtype == LQ_F32 ? 4 : 2);
        const bool wide = ysize % 16 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
        auto acc_free = [&](int b) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2)
                    mbar_arrive_peer(&acc_empty[b], 0);
                else
                    mbar_arrive(&acc_empty[b]);
            }
        };
        constexpr int COLS = T <= 32 ? 16 : T <= 64 ? 32 : 64;  // of a warp at a time
        constexpr int SIDES = S::OUT / 4, ROUNDS = (T + SIDES * COLS - 1) / (SIDES * COLS);
        const int quarter = warp & 3, side = warp >> 2;
        int j = 0;
        Fp4Tile t;
        for (int lin = first; lin < ntiles; lin += step) {
            if (!fp4_tile<S>(a, seg, lin, t)) continue;
            if (ok) ok = mbar_wait_cg<CG>(&acc_full[j & 1], (j >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const int nb = t.n0 + 128 * half + 32 * quarter, n = nb + lane;
            const uint32_t acc = tmem + (uint32_t(32 * quarter) << 16) + uint32_t((j & 1) * S::ACC_STEP);
            float* part = reinterpret_cast<float*>(smem);  // [T][128] sums of this CTA's share of K (split K: one tile a CTA)
#pragma unroll 1
            for (int i = 0; i < ROUNDS; ++i) {
                // The columns that the next tile's accumulator covers come first, and all of them to registers: the next tile's
                // MMAs wait for that, not for the stores.
                const int c0 = (S::ACC == 256 ? 128 * ((i + (j & 1) + 1) & 1) : SIDES * COLS * i) + COLS * side;
                if (c0 >= T) break;
                float v[COLS];
                uint32_t r[16];
#pragma unroll
                for (int c = 0; c < COLS; c += 16) {
                    uint32_t(&rr)[16] = *reinterpret_cast<uint32_t(*)[16]>(&v[c]);
                    tmem_ld_32x32b_x16(acc + c0 + c, rr);
                }
                tmem_wait_ld();
                if constexpr (S::STACK) {
#pragma unroll
                    for (int p = 1; p < P; ++p) {
                        tmem_ld_32x32b_x16(acc + p * T + c0, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 16; ++c) v[c] += __uint_as_float(r[c]);
                    }
                }
                if (S::ACC == 256 && i == 0) acc_free(0);
                if (S::ACC != 256 && i == ROUNDS - 1) acc_free(j & 1);
#pragma unroll
                for (int c = 0; c < COLS; c += 16) {
                    float(&u)[16] = *reinterpret_cast<float(*)[16]>(&v[c]);
                    if (CG == 1 && a.ks > 1) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) part[(c0 + c + q) * 128 + 32 * quarter + lane] = u[q];
                    } else {
                        if constexpr (S::KIND != FP4_SPLIT) {
#pragma unroll
                            for (int q = 0; q < 16; ++q) u[q] *= f.x;
                            if (f.y != 1.f) {
#pragma unroll
                                for (int q = 0; q < 16; ++q) u[q] *= f.y;
                            }
                        }
                        if (wide && nb + 32 <= a.N) {
                            if (t.r0 + c0 + c < t.r1) fp4_out16<S::TURN>(a, t, c0 + c, nb, u, stage + S::TURN * warp, lane);
                        } else {
#pragma unroll
                            for (int q = 0; q < 16; ++q) fp4_out<S>(a, t, c0 + c + q, n, u[q]);
                        }
                    }
                }
            }
            if (S::ACC != 256 && COLS * side >= T) acc_free(j & 1);  // (16 tokens: one warp a quarter reads)
            ++j;
        }
    }
    tc_fence_before();
    __syncwarp();
    if (CG == 1 && a.ks > 1) {
        // The CTAs of a cluster have one tile: each writes out the columns c with c % ks == its rank. Tensor memory is given back
        // before this one waits for the others' sums: held there, while another CTA of the cluster waits for its own, it could hold
        // up, and be held up by, a cluster of any kernel that does the same. (Between arriving and waiting, since all warps
        // together before it cost 0.2 us.)
        constexpr int readers = 32 * (S::OUT + 1);
        cluster_arrive();
        if (warp < S::OUT) named_arrive(1, readers);
        if (warp == FP4_OUT + 1) {
            named_barrier(1, readers);
            tc_fence_after();
            tc_dealloc<CG>(tmem, S::TMEM);
            __syncwarp();
        }
        cluster_wait();
        Fp4Tile t;
        if (warp < FP4_OUT && first < ntiles && fp4_tile<S>(a, seg, first, t)) {
            const float2 f = S::KIND == FP4_SPLIT ? make_float2(1.f, 1.f) : fp4_factors(a);
            const uint32_t part = smem_u32(smem) + lane * 16;  // a lane takes four rows of w
            for (int c = rank + a.ks * warp; c < T && t.r0 + c < t.r1; c += FP4_OUT * a.ks) {
                float4 p[8];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < a.ks) p[q] = ld_dsmem_f4(map_peer(part + c * 512, q));
                float4 v = p[0];
#pragma unroll
                for (int q = 1; q < 8; ++q)
                    if (q < a.ks) {
                        v.x += p[q].x;
                        v.y += p[q].y;
                        v.z += p[q].z;
                        v.w += p[q].w;
                    }
                if constexpr (S::KIND != FP4_SPLIT) v = make_float4(v.x * f.x * f.y, v.y * f.x * f.y, v.z * f.x * f.y, v.w * f.x * f.y);
                fp4_out4(a, t, c, t.n0 + 4 * lane, v);
            }
        }
        __syncwarp();
        cluster_sync();
        return;
    }
    if constexpr (CG == 2)
        cluster_sync();  // neither CTA leaves while the other's MMAs or arrivals may reach it
    else
        __syncthreads();
    if (warp == FP4_OUT + 1) {
        tc_fence_after();
        tc_dealloc<CG>(tmem, S::TMEM);
    }
}

// ---- activations of 16 bits in e4m3 pieces ---------------------------------------------------------

struct SplitArgs {
    const void* x;
    int64_t x_row;
    int rows, K, ktiles, nb, T, stack;  // stack: a token's pieces as rows of one scale tile
    bool vec;
    uint8_t* pieces;  // (P, rows, Kp)
    uint8_t* tiles;   // (token tile, K tile, nb, 512)
    const int32_t* order;  // gather > 0: row j is row order[j] / gather of x (order NULL: j / gather); 0: row j
    int gather, src_rows;
    int grouped, max_seg;
    const int32_t* starts;
    const int32_t* nseg;
};

// A warp takes 1,024 values of a row: the row's place is found once, four loads a lane are on their way together. (With a
// thread a group and its place searched at each, 16,004 gathered rows of 2,048 took 70 us.)
template <typename X, int P>
__global__ void __launch_bounds__(256) fp4_split_kernel(const SplitArgs a) {
    grid_dep_wait();
    grid_dep_launch();  // after the wait: the product reads weights ahead of this kernel's end
    const int lane = threadIdx.x & 31, words = fp4_padded(a.K) / 8, parts = (words + 127) / 128;
    const int64_t tasks = int64_t(a.rows) * parts;
    for (int64_t u = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; u < tasks; u += (int64_t(gridDim.x) * blockDim.x) >> 5) {
        const int row = int(u / parts), part = int(u - int64_t(row) * parts);
        int64_t src = row;
        if (a.gather) {
            const int pair = a.order ? a.order[row] : row;
            src = pair / a.gather;
            if (pair < 0 || src >= a.src_rows) {
                if (lane == 0) record_status(LQ_DEV_BOUNDS);
                src = -1;  // zeros
            }
        }
        Eight<X> v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int word = part * 128 + 32 * i + lane;
            v[i].zero();
            if (src >= 0 && word < words) v[i].load(static_cast<const X*>(a.x) + src * a.x_row, 8 * word, a.K, a.vec);
        }
        int tile = row / a.T, at = row % a.T;
        if (a.grouped) {
            int lo = a.starts ? 0 : row, hi = a.starts ? min(*a.nseg, a.max_seg) : 0;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (a.starts[mid] <= row) lo = mid; else hi = mid;
            }
            const int s0 = a.starts ? min(max(a.starts[lo], 0), row) : row;
            tile = s0 / a.T + lo + (row - s0) / a.T;
            at = (row - s0) % a.T;
        }
        const int tile_step = a.nb * 512;
        uint8_t *rowp[P], *scale[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int r = a.stack ? p * a.T + at : at, block = a.stack ? 0 : p * ((a.T + 127) / 128) + r / 128;
            rowp[p] = a.pieces + (int64_t(p) * a.rows + row) * (words * 8);
            scale[p] = a.tiles + int64_t(tile) * a.ktiles * tile_step + block * 512 + fp4_tile_byte(r % 128, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int word = part * 128 + 32 * i + lane;
            if (part * 128 + 32 * i >= words) break;  // (rows are a multiple of 16 words: half a warp may be beyond)
            uint2 piece[P];
            int byte[P];
            split8<X, P>(v[i], 0xFFFFFFFFu, piece, byte);
            if (word < words) {
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    *reinterpret_cast<uint2*>(rowp[p] + 8 * word) = piece[p];
                    if (word % 4 == 0) scale[p][(word >> 4) * tile_step + (word / 4 & 3)] = uint8_t(byte[p]);
                }
            }
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------

static int launch(const void* func, int grid, int threads, size_t smem, int cluster, cudaStream_t st, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(grid));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, func, args) == cudaSuccess ? LQ_OK : LQ_E_CUDA;
}

struct Fp4Call {
    const uint8_t* x;  // codes or pieces
    const uint8_t* xt;
    const uint32_t* w;
    const uint8_t* wt;
    int stack;         // experts, 1 for a dense product
    int64_t ttiles;    // most tiles of tokens that the call can have
    Fp4Args a;
};

// A matrix of bytes (or of packed 4-bit codes that TMA spreads to bytes), 128 of a row and `rows` rows a box.
static int map_rows(CUtensorMap* m, const void* base, bool spread, uint64_t row_bytes, uint64_t rows, uint32_t box_rows) {
    const uint64_t dims[2] = {spread ? 2 * row_bytes : row_bytes, rows}, str[1] = {row_bytes};
    const uint32_t box[2] = {128, box_rows};
    return make_tmap(m, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, str, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

// Scale tiles of 512 bytes, (outer, inner) of them; what a box has beyond the last is zeros.
static int map_scales(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint32_t box_inner, uint32_t box_outer) {
    const uint64_t dims[3] = {128, inner, outer}, str[2] = {512, 512 * inner};
    const uint32_t box[3] = {128, box_inner, box_outer};
    return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Clusters of ks CTAs that the current device runs at once: its SMs come in groups that a cluster does not leave, so that 48
// clusters of three need not fit 148 SMs. Asked once a device, kernel and size. (Of a kernel that allocates tensor memory the
// runtime counts one CTA an SM, whatever it allocates; narrow tiles run two, as their start times show.)
template <typename S>
static int max_clusters(int ks, size_t smem, int grouped) {
    static std::atomic<int> known[16][2][9];
    const int dev = device_info().device;
    if (dev < 0 || dev >= 16) return 0;
    std::atomic<int>& k = known[dev][grouped][ks];
    int n = k.load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(ks));
        cfg.blockDim = dim3(FP4_THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(ks);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, fp4_gemm_kernel<S>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        k.store(n > 0 ? n : -1, std::memory_order_relaxed);
    }
    return n;
}

template <typename S>
static int gemm_t(const Fp4Call& c, cudaStream_t st) {
    Fp4Args a = c.a;
    a.ns = (a.Kp + S::BK - 1) / S::BK;
    a.rtiles = (a.N + 127) / 128;
    Fp4Maps m = {};
    int rc = map_rows(&m.w, c.w, S::KIND == FP4_SPLIT, uint64_t(a.Kp) / 2, uint64_t(c.stack) * a.N, 128);
    if (!rc && !S::FUSE) rc = map_rows(&m.x, c.x, false, uint64_t(a.Kp) / (S::KIND == FP4_SPLIT ? 1 : 2), uint64_t(S::P) * a.M, S::T / S::CG);
    if (!rc) rc = map_scales(&m.ws, c.wt, a.ktiles, uint64_t(c.stack) * a.rtiles, S::KB, 1);
    if (!rc && !S::FUSE) rc = S::KIND == FP4_SPLIT ? map_scales(&m.xs, c.xt, S::NB, uint64_t(c.ttiles) * a.ktiles, S::NB, 1)
                                       : map_scales(&m.xs, c.xt, a.ktiles, (uint64_t(a.M) + 127) / 128, S::KB, S::NB);
    if (rc) return rc;
    const int sms = device_info().sm_count;
    a.ntn = (a.rtiles + S::CG - 1) / S::CG;
    const int64_t tiles = c.ttiles * a.ntn;
    if (tiles > INT32_MAX) return LQ_E_SHAPE;
    a.ntiles = int(tiles);
    a.nst = S::stages(a.grouped);
    const size_t smem = S::beside(a.grouped) + size_t(a.nst) * S::STAGE;
    static_assert(S::ACC == 256 || S::T * 512 <= S::stages(true) * S::STAGE, "the partial sums of a split fit the ring");
    auto kern = fp4_gemm_kernel<S>;
    // The same limit at every call: set to the call's own size, a dense call on one host thread lowered it between a grouped call's
    // setting and its launch on another, which was then refused.
    constexpr size_t dense = S::beside(false) + size_t(S::stages(false)) * S::STAGE, grouped = S::beside(true) + size_t(S::stages(true)) * S::STAGE;
    constexpr int limit = int(dense > grouped ? dense : grouped);
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, limit) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
        return LQ_E_CUDA;
    // Few tiles: a tile's K split over as many CTAs of a cluster as still run all at once, each with a stage at least.
    a.ks = 1;
    if (S::CG == 1) {
        const int most = a.ns < 8 ? a.ns : 8;
        for (int ks = most; ks > 1 && a.ks == 1; --ks)
            if (tiles * ks <= int64_t(sms) * (S::T <= 32 ? 2 : 1) && tiles <= max_clusters<S>(ks, smem, a.grouped) * (S::T <= 32 ? 2 : 1)) a.ks = ks;
    }
    const int64_t slots = int64_t(sms) * (S::T <= 32 ? 2 : 1);
    const int64_t grid = S::CG == 2 ? (tiles < sms / 2 ? tiles : sms / 2) * 2 : a.ks > 1 ? tiles * a.ks : tiles < slots ? tiles : slots;
    void* args[] = {&m, &a};
    return launch(reinterpret_cast<const void*>(kern), int(grid), FP4_THREADS, smem, S::CG == 2 ? 2 : a.ks, st, args);
}

template <int KIND, int P, typename X = void>
static int gemm_tokens(const Fp4Call& c, int T, bool fuse, cudaStream_t st) {
    if constexpr (KIND == FP4_SPLIT)
        if (fuse) return T == 16 ? gemm_t<Fp4Shape<KIND, P, 16, 1, X>>(c, st) : gemm_t<Fp4Shape<KIND, P, 32, 1, X>>(c, st);
    switch (T) {
        case 16: return gemm_t<Fp4Shape<KIND, P, 16>>(c, st);
        case 32: return gemm_t<Fp4Shape<KIND, P, 32>>(c, st);
        case 64: return gemm_t<Fp4Shape<KIND, P, 64>>(c, st);
        case 128:  // enough tiles for all SMs: pairs; else one CTA a tile, or several that split its K
            if (c.ttiles * ((c.a.N + 255) / 256) * 2 >= device_info().sm_count) return gemm_t<Fp4Shape<KIND, P, 128, 2>>(c, st);
            return gemm_t<Fp4Shape<KIND, P, 128>>(c, st);
        default: return gemm_t<Fp4Shape<KIND, P, 256, 2>>(c, st);
    }
}

// Tokens a tile. (A product of both in 4 bits has scale tiles of 128 tokens, so narrower tiles only where one holds them all.)
// Beyond 128 tokens tiles of 256 read the weights half as often as tiles of 128, which in turn end closer to the last token: 256 but
// where that adds an eighth of tokens or more. Both ways, 16 bits by 14336 x 4096: 256 tokens 31 us in tiles of 256 and 33 of 128, 300
// tokens 51 and 44, 600 71 and 58, 1,200 101 and 116, 2,048 183 and 189. The rule does not count tiles, and where weights have
// few rows pairs of CTAs leave SMs idle: 256 tokens by 2560 x 9728 take 53 us, 25 in tiles of 128; 512 by 4096 x 4096 39 and 29.
static int tile_tokens(int rows) {
    if (rows <= 128) return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const int64_t narrow = (int64_t(rows) + 127) / 128 * 128, wide = (int64_t(rows) + 255) / 256 * 256;
    return wide * 8 <= narrow * 9 ? 256 : 128;
}

int fp4_qmm_run(const uint32_t* xc, const uint8_t* xt, const float* xf, const uint32_t* wc, const uint8_t* wt, const float* wf,
                int M, int N, int K, int mode, int glu, int dtype, void* y, cudaStream_t st) {
    Fp4Call c = {};
    const int T = tile_tokens(M);
    c.x = reinterpret_cast<const uint8_t*>(xc);
    c.w = wc;
    c.stack = 1;
    Fp4Args& a = c.a;
    a.M = M;
    a.N = N;
    a.Kp = fp4_padded(K);
    a.ktiles = fp4_ktiles(K, mode);
    c.ttiles = (M + T - 1) / T;
    a.glu = glu;
    a.dtype = dtype;
    c.wt = wt;
    c.xt = xt;
    a.xf = xf;
    a.wf = wf;
    a.y = y;
    return mode == LQ_MXFP4 ? gemm_tokens<FP4_MX, 1>(c, T, false, st) : gemm_tokens<FP4_NV, 1>(c, T, false, st);
}

// Token tiles of the rows of a call (grouped: one number a segment may go unused), and the bytes of the split's results.
static int64_t split_tiles(int rows, int T, int segments) { return segments ? rows / T + segments : (rows + T - 1) / T; }
static int split_blocks(int P, int T) { return T <= 32 ? 1 : P * ((T + 127) / 128); }
static size_t split_pieces_bytes(int rows, int K, int P) { return (size_t(P) * rows * fp4_padded(K) + 511) / 512 * 512; }

// Tokens a tile of rows that are dealt out to segments: twice the average, so that most segments are one tile; long segments
// have tiles of 128, whose last is half as wide (64 experts, 250 rows each: 143 us in tiles of 256, 110 of 128, for 4,001 tokens'
// gate and up), until that is a small part of them (8 experts: 250 rows each 26 and 27 us, 1,000 59 and 65, 2,000 112 and 119).
static int grouped_tokens(int rows, int segments, int max_rows) {
    const int64_t average = int64_t(rows) / (segments > 0 ? segments : 1), want = 2 * average;
    const int T = tile_tokens(int(want < max_rows ? want : max_rows));
    return T > 128 && average < 1024 ? 128 : T;
}

// Whether the product makes the pieces of x itself: few tokens, and all tiles run at once.
static bool fused(int T, int64_t ttiles, int N) { return T <= 32 && ttiles * ((N + 127) / 128) <= 2 * int64_t(FP4_FUSE_SMS); }

// Pieces of a value: two hold the 8 bits of bf16, three the 11 of fp16 (and 14 or more of 32 bits).
static int fp4_pieces(int x_dtype) { return x_dtype == LQ_BF16 ? 2 : 3; }

size_t fp4_linear_workspace_bytes(int rows, int N, int K, int x_dtype, int segments, int max_rows) {
    const int P = fp4_pieces(x_dtype), T = segments ? grouped_tokens(rows, segments, max_rows) : tile_tokens(rows);
    if (fused(T, split_tiles(rows, T, segments), N)) return 0;
    return split_pieces_bytes(rows, K, P) +
           size_t(split_tiles(rows, T, segments)) * fp4_ktiles(K, LQ_MXFP4) * split_blocks(P, T) * 512;
}

int fp4_linear_run(const Fp4Linear& l, cudaStream_t st) {
    const int P = fp4_pieces(l.x_dtype);
    const int T = l.segments ? grouped_tokens(l.rows, l.segments, l.max_rows) : tile_tokens(l.rows);
    if (l.ws_bytes < fp4_linear_workspace_bytes(l.rows, l.N, l.K, l.x_dtype, l.segments, l.max_rows)) return LQ_E_SHAPE;
    uint8_t* ws = static_cast<uint8_t*>(l.ws);
    SplitArgs s = {};
    s.ktiles = fp4_ktiles(l.K, LQ_MXFP4);
    const bool vec = aligned(l.x, 16) && l.x_row % (l.x_dtype == LQ_F32 ? 4 : 8) == 0;
    const bool fuse = fused(T, split_tiles(l.rows, T, l.segments), l.N);
    if (!fuse) {
        s.x = l.x;
        s.x_row = l.x_row;
        s.rows = l.rows;
        s.K = l.K;
        s.nb = split_blocks(P, T);
        s.T = T;
        s.stack = T <= 32;
        s.vec = vec;
        s.pieces = ws;
        s.tiles = ws + split_pieces_bytes(l.rows, l.K, P);
        s.order = l.order;
        s.gather = l.gather;
        s.src_rows = l.src_rows;
        s.grouped = l.segments > 0;
        s.max_seg = l.segments;
        s.starts = l.starts;
        s.nseg = l.nseg;
        const int64_t units = int64_t(l.rows) * ((fp4_padded(l.K) + 1023) / 1024);  // of a warp
        const int64_t most = int64_t(device_info().sm_count) * 8, blocks = (units + 7) / 8;
        const void* split = l.x_dtype == LQ_BF16  ? reinterpret_cast<const void*>(fp4_split_kernel<__nv_bfloat16, 2>)
                            : l.x_dtype == LQ_F16 ? reinterpret_cast<const void*>(fp4_split_kernel<__half, 3>)
                                                  : reinterpret_cast<const void*>(fp4_split_kernel<float, 3>);
        void* sargs[] = {&s};
        const int rc = launch(split, int(blocks < most ? blocks : most), 256, 0, 1, st, sargs);
        if (rc) return rc;
    }
    Fp4Call c = {};
    c.x = s.pieces;
    c.w = l.wc;
    c.stack = l.segments ? l.E : 1;
    Fp4Args& a = c.a;
    a.M = l.rows;
    a.N = l.N;
    a.Kp = fp4_padded(l.K);
    a.ktiles = s.ktiles;
    c.ttiles = split_tiles(l.rows, T, l.segments);
    a.glu = l.glu;
    a.dtype = l.dtype;
    a.piece_rows = l.rows;
    a.x_rows = l.x;
    a.x_row = l.x_row;
    a.K = l.K;
    a.vec = vec;
    a.order = l.order;
    a.gather = l.gather;
    a.src_rows = l.src_rows;
    c.wt = l.wt;
    c.xt = s.tiles;
    a.y = l.y;
    a.grouped = l.segments > 0;
    a.E = l.E;
    a.starts = l.starts;
    a.experts = l.experts;
    a.nseg = l.nseg;
    a.max_seg = l.segments;
    if (l.x_dtype == LQ_BF16) return gemm_tokens<FP4_SPLIT, 2, __nv_bfloat16>(c, T, fuse, st);
    if (l.x_dtype == LQ_F16) return gemm_tokens<FP4_SPLIT, 3, __half>(c, T, fuse, st);
    return gemm_tokens<FP4_SPLIT, 3, float>(c, T, fuse, st);
}

}  // namespace lq
