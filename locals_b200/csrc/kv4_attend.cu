// Attention of queries over a paged 4-bit cache (layout: kv4.cuh).
//
// Query i of request b stands at position lens[b] - new[b] + i and sees the keys from max(0, position - window + 1)
// (window 0: from 0) to its own: out = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)), s_j = scale q . k_j,
// and 0 where nothing is seen.
//
// kv4_attend_kernel. The rows of a (request, kv head) are its queries times the G query heads of the kv head; a tile of 8 NT
// of them is the n side of m16n8k16 fp16 MMAs whose m side is 16 keys (scores, S^T = K Q^T) or 16 dimensions (values,
// O^T = V^T P^T), so that few rows fill the MMA and each key is unpacked once for all of them. The 4-bit codes enter the
// MMA as fp16 subnormals, with no arithmetic at all: a word's bits & 0x000f000f are the pair (code 0, code 4) * 2^-24,
// & 0x00f000f0 the pair (code 1, code 5) * 2^-20, and the same of word >> 8; every product of them is exact in the fp32
// accumulator. What differs between the nibble's places is put right on the other side: queries that meet 2^-20 codes are
// divided by 16 beforehand, output dimensions that they made are afterwards. The groups' scales and biases never touch the
// key codes:
//   s_j = scale * sum_g ks_jg (q . codes)_g + kb_jg sum(q)_g,
//   o_g = sum_j w_jg (codes_jg - z_jg) + p_j (vb_jg + z_jg vs_jg),   w_jg = p_j vs_jg,  z_jg = round(-vb_jg / vs_jg) in 0..15.
// Scores, softmax statistics and outputs are fp32. Two roundings to fewer bits:
//   queries to fp16 after a power of two a row that puts its largest at 2^13 .. 2^14: exact for fp16 and bf16 but for
//     values 2^-27 below the row's largest. A row by itself: the tile holds other heads and other tokens of the request;
//   w to fp16 (2^-11 against the 2^-8 of a bf16 output; an fp16 output's error grows from 2.0e-4 to 2.2e-4 by it), after a
//     power of two a row that puts the largest value scale that the row has seen at 2^5 .. 2^10 (vf for the warp, a row's
//     difference from it, xl, in its probabilities): values are held to 2^-30 of the largest that the row sees. codes - z
//     (exact on subnormals, one packed subtraction a pair) takes out of a group what its codes and its bias have in common,
//     so that this is a rounding of the value itself, however near to 0 it lies.
// A score tile's accumulator layout is transposed into the value MMA's operand by movmatrix. The running maximum of a row is
// only followed when it has grown by 2^4, so that most steps rescale nothing.
// A key's scales and biases become floats once a step, one key a lane, and go to its reads through shared memory. A masked
// key's score is -inf; a key without a page has none; a key whose values are not finite has zero values and a NaN key, so
// that what a place holds reaches only the rows that see it.
//
// Each warp walks 32-key steps through a ring of its own, filled with cp.async STAGES - 1 steps ahead; the pages of the
// next 8 steps are looked up by the 32 lanes at once (8 keys always lie in one page). Rows are permuted within a chunk
// (P8) and 32-byte pieces swizzled (kv4_swz) so that every shared load is free of bank conflicts.
// The keys of all (request, kv head, tile)s, in steps of 128, are dealt out evenly over one wave of CTAs, wherever the boundaries
// fall; a CTA that holds only part of an item writes a part (m, l, O) to the workspace, at most two a CTA, and
// kv4_join_kernel joins each divided item. Where every item can have a cluster of CTAs and few steps (kv4_cluster), the
// cluster's CTAs share the item and join through distributed shared memory: one launch.
//
// What bounds it. The bytes are (D + D / 8) a key and kv head (144 at D = 128); the instructions are about 730 a warp and 32
// keys (unpacking 200, z 64, MMAs 48, the rest loads, scales and softmax), and they are what the time goes to: 2.3 a clock
// and SM, the ALU pipe 47% busy, tensor pipe 21%: no pipe is full, a step's chain (scales, z, scores, maximum, exponentials,
// values) waits on itself. Measured, GPU time of a call: 4 requests of 131,072 keys, 32 heads on 4, D = 128, fp16: 81.9 us =
// 3.69 TB/s (56% of the copy rate); 64 requests of up to 8,191 keys, 32 heads on 4, bf16: 54.6 us = 2.83 TB/s; one request of
// 1,001 keys: 6.9 us among others (launch, one pass of dependent loads, two cluster barriers). A power of two a row, for the
// queries and for the values, is 0.6 us of that, 1.2 of 54.6 and 2.4 of 81.9.
// Tried and slower: 4 CTAs a SM at 128 registers (89.6 against 83.3 us, it spills), 5 (126); a ring of 2 stages is as fast
// as 3 at D = 128.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "kv4_attend.cuh"
#include "lq_host.h"
#include "lq_ptx.cuh"
#include "lq_status.cuh"

namespace lq {

constexpr int KV4_NW = 4;                 // warps a CTA
constexpr int KV4_KEYS = 32;              // keys a warp step
constexpr int KV4_STEP = KV4_NW * KV4_KEYS;  // keys a CTA step
__device__ __forceinline__ uint32_t kv4_cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// What an item costs beside its steps (pages and queries fetched, the ring filled, the warps joined), in steps. 64 requests
// of up to 8,191 keys: 1: 69 us, 2: 63, 4 to 7: 56.
constexpr int KV4_ITEM = 5;

__device__ __forceinline__ Kv4Req kv4_request(const Kv4AttArgs& a, int b) {
    Kv4Req r = kv4_new(a, b);
    if (r.fresh * a.G > a.split_rows) r.fresh = 0;  // (kv4_prefill's)
    const long long room = (long long)a.width * a.pool.page;
    const int keys = int(min((long long)max(r.len, 0), room));
    const int lo = a.window ? max(0, r.len - r.fresh + 1 - a.window) : 0;
    r.s_lo = min(lo, keys) / KV4_STEP;
    r.s_hi = max((keys + KV4_STEP - 1) / KV4_STEP, r.s_lo + 1);  // (a step at least: what sees nothing is written too)
    return r;
}

// Items of a request: its kv heads' tiles of R rows, a kv head's side by side (they read the same keys).
template <int R>
__device__ __forceinline__ int kv4_items(const Kv4AttArgs& a, const Kv4Req& r) {
    return (r.fresh * a.G + R - 1) / R * a.pool.KVH;
}

// Units of all of request b's items.
template <int R>
__device__ __forceinline__ int kv4_weight(const Kv4AttArgs& a, int b) {
    if (b >= a.B) return 0;
    const Kv4Req r = kv4_request(a, b);
    return r.fresh ? (r.steps() + KV4_ITEM) * kv4_items<R>(a, r) : 0;
}

// Inclusive sum over the CTA's 128 threads, and their total.
__device__ __forceinline__ int kv4_scan(int v, int* red, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    __syncthreads();  // (red may still be read from before)
    if (lane == 31) red[warp] = v;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int k = 0; k < KV4_NW; ++k) {
        if (k == warp) v += sum;
        sum += red[k];
    }
    *total = sum;
    return v;
}

template <int D>
struct Kv4Shape {
    static constexpr int GR = D / 64;
    static constexpr int RB = D / 2;                      // bytes of codes a key
    static constexpr int KV_BYTES = KV4_KEYS * RB;        // a step's key (or value) codes
    static constexpr int SC = 8 * GR;                     // bytes of scales and biases a key
    static constexpr int STAGE = 2 * KV_BYTES + KV4_KEYS * SC;
    static constexpr int STAGES = D == 64 ? 4 : D == 128 ? 3 : 2;
    static constexpr int FL = 4 * GR;                     // floats a key made of its scales and biases
    static constexpr int ZB = 2 * GR;                     // bytes of z a key
    static constexpr int WARP = STAGES * STAGE + KV4_KEYS * (FL * 4 + ZB);
    static constexpr int RING = KV4_NW * WARP;            // 39,168 / 59,904 / 82,944 bytes: 4, 3, 2 CTAs a SM
};

// Row x of a chunk's 8 keys in the MMA's order, and the 32-byte piece of group g in row r: with these, the 4 rows that
// half a warp reads as keys, and the 4 that a warp reads as values, fall on different banks.
__device__ __forceinline__ int kv4_p8(int x) { return (0x57463120u >> (4 * x)) & 7; }
__device__ __forceinline__ int kv4_p8_inv(int r) { return (0x64753120u >> (4 * r)) & 7; }
template <int D>
__device__ __forceinline__ int kv4_swz(int r, int g) {
    return D == 64 ? 0 : D == 128 ? (g ^ ((r >> 1) & 1)) : (g ^ (r & 3));
}

// a - b on pairs of fp16 subnormals: exact.
__device__ __forceinline__ uint32_t kv4_sub(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// N floats from shared memory: from a multiple of 16 bytes where N is above 3, of 8 else.
template <int N>
__device__ __forceinline__ void kv4_floats(uint32_t addr, float (&f)[N]) {
    constexpr int Q = N / 4 * 4;
#pragma unroll
    for (int i = 0; i < Q; i += 4)
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(f[i]), "=f"(f[i + 1]), "=f"(f[i + 2]), "=f"(f[i + 3])
                     : "r"(addr + 4 * i));
    if constexpr (N % 4 >= 2) asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(f[Q]), "=f"(f[Q + 1]) : "r"(addr + 4 * Q));
    if constexpr (N % 2 == 1) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[N - 1]) : "r"(addr + 4 * (N - 1)));
}

// CTAs a SM, by registers (8 rows: 128 / 168 / 255 a thread) and shared memory.
constexpr int kv4_resident(int D, int NT) { return NT == 2 || D == 256 ? 2 : D == 128 ? 3 : 4; }

// CL: one cluster of CTAs an item, each with a run of its steps, joined through distributed shared memory instead of the
// workspace and a second launch.
template <typename T, int D, int NT, bool CL>
__global__ void __launch_bounds__(KV4_NW * 32, kv4_resident(D, NT)) kv4_attend_kernel(const Kv4AttArgs a) {
    using S = Kv4Shape<D>;
    constexpr int GR = S::GR, R = 8 * NT;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    __shared__ int red[KV4_NW], found[2];
    grid_dep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, c = lane & 3;
    const int tid = threadIdx.x, KVH = a.pool.KVH, G = a.G;

    kv4_zero_rest(a, D);

    int b = 0, n = 0;
    long long at = 0, total = 0, x0 = 0, x1 = 1;  // steps before request b; of all; this CTA's
    int32_t* rec = a.records + blockIdx.x * 8;    // what the join kernel does for this CTA's first step
    if constexpr (!CL) {
        // ---- this CTA's share of the steps: requests are scanned 128 at a time ----
        const int w0 = kv4_weight<R>(a, tid);
        int sum0;
        const int s0 = kv4_scan(w0, red, &sum0);
        total = sum0;
        for (int b0 = KV4_NW * 32; b0 < a.B; b0 += KV4_NW * 32) {
            int sum;
            kv4_scan(kv4_weight<R>(a, b0 + tid), red, &sum);
            total += sum;
        }
        n = int(min((long long)gridDim.x, total));  // (every CTA below n has a step, those above none)
        if (tid == 0) rec[0] = 0;
        if (int(blockIdx.x) >= n) return;
        x0 = (long long)blockIdx.x * total / n, x1 = ((long long)blockIdx.x + 1) * total / n;
        for (int b0 = 0;; b0 += KV4_NW * 32) {
            int sum = sum0, s = s0, w = w0;
            if (b0) {
                w = kv4_weight<R>(a, b0 + tid);
                s = kv4_scan(w, red, &sum);
            }
            if (at + sum <= x0) {
                at += sum;
                continue;
            }
            if (at + s > x0 && at + s - w <= x0) found[0] = b0 + tid, found[1] = s - w;  // one thread's
            __syncthreads();
            b = found[0];
            at += found[1];
            break;
        }
    }

    const uint32_t ring = smem_u32(kv4_smem) + warp * S::WARP;
    const uint32_t made = ring + S::STAGES * S::STAGE;  // the step's floats: ks', kb, vs', vb' (GR each) a key
    const uint32_t zeds = made + KV4_KEYS * S::FL * 4;  // and its z, 2 bytes each: (group, chunk, place in the MMA's order)
    // places in a stage that this lane reads: keys p8(gid) (+ 8) of a chunk and its floats, values p8(2c), p8(2c + 1) (+ 8)
    uint32_t k_at[GR], va_at[GR], vb_at[GR];
#pragma unroll
    for (int g = 0; g < GR; ++g) {
        k_at[g] = kv4_p8(gid) * S::RB + (kv4_swz<D>(kv4_p8(gid), g) << 5) + 8 * c;
        va_at[g] = S::KV_BYTES + kv4_p8(2 * c) * S::RB + (kv4_swz<D>(kv4_p8(2 * c), g) << 5) + 4 * gid;
        vb_at[g] = S::KV_BYTES + kv4_p8(2 * c + 1) * S::RB + (kv4_swz<D>(kv4_p8(2 * c + 1), g) << 5) + 4 * gid;
    }
    const uint32_t f_at = made + kv4_p8(gid) * S::FL * 4;
    // this lane's place of z: key lane
    const uint32_t z_at = zeds + (lane >> 4) * 32 + (kv4_p8_inv(lane & 7) >> 1) * 8 + ((lane >> 3) & 1) * 4 + (kv4_p8_inv(lane & 7) & 1) * 2;

    long long x = x0;
    while (x < x1) {
        int item, st0, st1;  // the request's item: kv head, tile
        if constexpr (CL) {
            const int per = KVH * ((a.split_rows + R - 1) / R);
            item = int(blockIdx.x / kv4_cluster_size());
            b = item / per;
            item -= b * per;
        }
        const Kv4Req rq = kv4_request(a, b);
        const int items = kv4_items<R>(a, rq), tiles = items / KVH;
        if constexpr (CL) {
            st0 = rq.steps() * int(cluster_ctarank()) / int(kv4_cluster_size());
            st1 = rq.steps() * int(cluster_ctarank() + 1) / int(kv4_cluster_size());
            x = x1;
            if (item >= items) return;  // (the whole cluster)
        } else {
            const int units = rq.steps() + KV4_ITEM;
            item = int((x - at) / units);
            if (!rq.fresh || item >= items) {  // on to the next request
                if (rq.fresh) at += (long long)units * items;
                ++b;
                continue;
            }
            const long long item_at = at + (long long)item * units;
            const int u1 = int(min((long long)units, x1 - item_at));
            st0 = max(int(x - item_at) - KV4_ITEM, 0), st1 = max(u1 - KV4_ITEM, 0);
            x = item_at + u1;
            if (st0 == st1) continue;
            if (st0 > 0 && tid == 0) {  // (only a CTA's first item can begin before it)
                const long long key0 = item_at + KV4_ITEM;
                rec[1] = rq.first;
                rec[2] = min(rq.fresh * G - item % tiles * R, R);
                rec[3] = item / tiles;
                rec[5] = item % tiles * R;
                rec[4] = kv4_owner(key0 + rq.steps() - 1, total, n);
                rec[0] = kv4_owner(key0, total, n) == int(blockIdx.x) - 1;  // the first boundary within its item
            }
        }
        const int kvh = item / tiles, row0 = (item - kvh * tiles) * R, rows = min(rq.fresh * G - row0, R);
        // what the rows see: keys below hi_max, from lo_min on; all of them see [lo_max, hi_min)
        const int base = rq.len - rq.fresh;  // position of query 0
        const int p0 = base + row0 / G, p1 = base + (row0 + rows - 1) / G;  // of the first and the last row
        const int room = int(min((long long)a.width * a.pool.page, 0x7fffffffLL));
        if (rq.len > room) record_status(LQ_DEV_BOUNDS);
        const int hi_min = min(p0 + 1, room), hi_max = min(p1 + 1, room);
        const int lo_min = a.window ? max(p0 + 1 - a.window, 0) : 0, lo_max = a.window ? max(p1 + 1 - a.window, 0) : 0;
        const int k_lo = max((rq.s_lo + st0) * KV4_STEP, lo_min / KV4_KEYS * KV4_KEYS);
        const int k_hi = min((rq.s_lo + st1) * KV4_STEP, hi_max);
        // this warp's 32-key steps: first, first + 128, ...
        const int first = ((k_lo + KV4_STEP - 1 - warp * KV4_KEYS) / KV4_STEP) * KV4_STEP + warp * KV4_KEYS;
        const int steps = k_hi > first ? (k_hi - first + KV4_STEP - 1) / KV4_STEP : 0;

        // lane l's page lookup: run l & 3 (of 8 keys) of step t0 + (l >> 2); row 0 where there is none. miss: bit l, some row
        // sees the run but it has no page (what lies behind a window may have been freed)
        auto lookup = [&](int t0, uint32_t* miss) -> uint32_t {
            const int key = first + (t0 + (lane >> 2)) * KV4_STEP + (lane & 3) * 8;
            uint32_t row = 0;
            bool gone = false;
            if (t0 + (lane >> 2) < steps && key < hi_max && key + 8 > lo_min) {
                const int pg = key / a.pool.page, id = a.table[(size_t)b * a.width + pg];
                gone = unsigned(id) >= unsigned(a.pool.pages);
                if (gone)
                    record_status(LQ_DEV_BOUNDS);
                else
                    row = kv4_row(a.pool, id, kvh, key - pg * a.pool.page);
            }
            *miss = __ballot_sync(0xffffffffu, gone);
            return row;
        };
        uint32_t miss_now, miss_next, miss_issued;  // of the steps computed, looked up, and issued
        uint32_t runs = lookup(0, &miss_now), runs_next = lookup(8, &miss_next);
        miss_issued = miss_now;

        // ---- the ring: a step's codes, scales and biases into its stage (a run without a page reads row 0, unused) ----
        auto issue = [&](int t, uint32_t sb) {
            constexpr int PIECES = S::RB / 16;  // 16-byte pieces a key
            constexpr int J = KV4_KEYS * PIECES / 32;
            const int sel = (t & 7) * 4;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int e = lane + 32 * j, r = e / PIECES, p = e % PIECES;
                const size_t from = size_t(__shfl_sync(0xffffffffu, runs, sel + r / 8)) * S::RB + (r & 7) * S::RB + p * 16;
                const uint32_t off = r * S::RB + (kv4_swz<D>(r, p >> 1) << 5) + ((p & 1) << 4);
                cp_async(sb + off, reinterpret_cast<const uint8_t*>(a.pool.kq) + from, 16, true);
                cp_async(sb + S::KV_BYTES + off, reinterpret_cast<const uint8_t*>(a.pool.vq) + from, 16, true);
            }
            // scales and biases: a key's four arrays side by side (two keys' for one group: a pair of 2-byte values)
            constexpr int PK = D == 64 ? 2 : 1, BY = D == 256 ? 8 : 4;
            const int r = (lane % (KV4_KEYS / PK)) * PK;
            const size_t row = size_t(__shfl_sync(0xffffffffu, runs, sel + r / 8) + (r & 7)) * GR;
            const uint32_t dst = sb + 2 * S::KV_BYTES + r * S::SC;
            if (D != 64 || lane < 16) {
                cp_async(dst, a.pool.ks + row, BY, true);
                cp_async(dst + BY, a.pool.kb + row, BY, true);
                cp_async(dst + 2 * BY, a.pool.vs + row, BY, true);
                cp_async(dst + 3 * BY, a.pool.vb + row, BY, true);
            }
        };
        auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
#pragma unroll
        for (int t = 0; t < S::STAGES - 1; ++t) {
            if (t < steps) issue(t, ring + t * S::STAGE);
            commit();
        }

        // ---- queries: fp16 B fragments times a row's power of two, and the group sums of what the MMA sees ----
        // (2^24 of the codes: 2^12 with the scales, 2^12 with the row's factor alpha, so that neither leaves its range)
        uint32_t qb[NT][GR][2][2][2];
        float qs[NT][GR][2], alpha[NT][2];
        {
            uint4 raw[NT][GR][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = 8 * t + gid, qi = (row0 + row) / G;
                const uint4* src = reinterpret_cast<const uint4*>(a.q + ((size_t)(rq.first + qi) * a.H + kvh * G + row0 + row - qi * G) * D);
#pragma unroll
                for (int g = 0; g < GR; ++g)
#pragma unroll
                    for (int u = 0; u < 2; ++u) raw[t][g][u] = row < rows ? src[8 * g + 2 * c + u] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float mx = 0.0f;  // of row gid: its four lanes'
#pragma unroll
                for (int g = 0; g < GR; ++g)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[t][g][u]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mx = fmaxf(mx, fmaxf(fabsf(F16Traits<T>::to_f32(w[i] & 0xffffu)),
                                                 fabsf(F16Traits<T>::to_f32(w[i] >> 16))));
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                // 2^E with the largest |q| at 2^13 .. 2^14
                const int E = mx > 0.0f ? min(13 - (int(__float_as_uint(mx) >> 23) - 127), 126) : 0;
                const float f = __uint_as_float(uint32_t(127 + E) << 23);
                const float back = a.scale_log2 * __uint_as_float(uint32_t(127 + 12 - E) << 23);
#pragma unroll
                for (int e = 0; e < 2; ++e) alpha[t][e] = __shfl_sync(0xffffffffu, back, (2 * c + e) * 4);
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    float sum = 0.0f;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[t][g][u]);
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[2 * i] = __half2float(__float2half_rn(F16Traits<T>::to_f32(w[i] & 0xffffu) * f));
                            v[2 * i + 1] = __half2float(__float2half_rn(F16Traits<T>::to_f32(w[i] >> 16) * f));
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum += v[i];
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            qb[t][g][u][m][0] = cvt_f16x2(v[2 * m + 4], v[2 * m]);
                            qb[t][g][u][m][1] = cvt_f16x2(v[2 * m + 5] * 0.0625f, v[2 * m + 1] * 0.0625f);
                        }
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                    for (int e = 0; e < 2; ++e)  // this lane's columns 2c + e of the score tile
                        qs[t][g][e] = 0x1p-12f * __shfl_sync(0xffffffffu, sum, (2 * c + e) * 4);
                }
            }
        }

        float o[NT][4 * GR][4], hb[NT][GR][2], m[NT][2], l[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int i = 0; i < 4 * GR; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) o[t][i][u] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[t][e] = -INFINITY, l[t][e] = 0.0f;
#pragma unroll
                for (int g = 0; g < GR; ++g) hb[t][g][e] = 0.0f;
            }
        }
        float vf = 1.0f;       // the value scales' power of two: 2^(132 - e0), for a largest scale whose exponent bits are e0
        int e0 = 0;
        float xl[NT][2];       // and a column's beyond it: p and l are 2^xl times as large (negative: it has seen none yet)
        uint32_t v_limit = 0;  // bits of the least value scale that some column's power does not fit
#pragma unroll
        for (int t = 0; t < NT; ++t) xl[t][0] = xl[t][1] = -1.0f;
        // o and hb by f0 (even columns) and f1
        auto rescale = [&](int t, float f0, float f1) {
#pragma unroll
            for (int i = 0; i < 4 * GR; ++i) {
                o[t][i][0] *= f0;
                o[t][i][1] *= f1;
                o[t][i][2] *= f0;
                o[t][i][3] *= f1;
            }
#pragma unroll
            for (int g = 0; g < GR; ++g) hb[t][g][0] *= f0, hb[t][g][1] *= f1;
        };

        // Column 8 t + 2 c + e's keys: [lo, hi).
        auto column = [&](int t, int e, int* lo, int* hi) {
            const int end = base + (row0 + min(8 * t + 2 * c + e, rows - 1)) / G + 1;
            *hi = min(end, room), *lo = a.window ? max(end - a.window, 0) : 0;
        };
        auto partly = [&](int key0, uint32_t miss) { return key0 < lo_max || key0 + KV4_KEYS > hi_min || miss; };
        // Fits the columns' powers of two to the scales that they see in a step (bits: the largest; top: this lane's key's):
        // one that grows leaves its limit at once, to 2^5 .. 2^6, the others stay as they are.
        auto fit = [&](uint32_t bits, float top, int key0) {
            int ce[NT][2], seen[NT][2], most = 0;  // exponent bits: that a column is fitted to (0: none yet), of what it sees
#pragma unroll
            for (int t = 0; t < NT; ++t) seen[t][0] = seen[t][1] = int(bits >> 23);
            if (p0 != p1 && partly(key0, 0)) {  // (what no row sees is 0 in top)
                int lo[NT][2], hi[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) column(t, e, &lo[t][e], &hi[t][e]), seen[t][e] = -1;
#pragma unroll 4
                for (int k = 0; k < KV4_KEYS; ++k) {
                    const int x = int(__shfl_sync(0xffffffffu, __float_as_uint(top), k) >> 23);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (key0 + k >= lo[t][e] && key0 + k < hi[t][e]) seen[t][e] = max(seen[t][e], x);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    ce[t][e] = xl[t][e] < 0.0f ? 0 : e0 - int(xl[t][e]);
                    if (seen[t][e] >= (ce[t][e] ? ce[t][e] + 5 : 0)) ce[t][e] = max(seen[t][e], 64);  // (at least 2^-63)
                    most = max(most, ce[t][e]);
                }
            const int e1 = int(__reduce_max_sync(0xffffffffu, unsigned(most)));
            int least = 255;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float f[2] = {1.0f, 1.0f};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (ce[t][e]) ce[t][e] = max(ce[t][e], e1 - 100);
                    least = min(least, ce[t][e]);
                    if (xl[t][e] >= 0.0f) {
                        const int was = e0 - int(xl[t][e]), grows = (e1 - ce[t][e]) - int(xl[t][e]);
                        f[e] = __uint_as_float(uint32_t(max(127 + was - ce[t][e], 1)) << 23);
                        l[t][e] *= __uint_as_float(uint32_t(127 + grows) << 23);
                    }
                    if (ce[t][e]) xl[t][e] = float(e1 - ce[t][e]);
                }
                rescale(t, f[0], f[1]);
            }
            e0 = e1;
            if (e1) vf = __uint_as_float(uint32_t(127 + 132 - e1) << 23);
            least = int(__reduce_min_sync(0xffffffffu, unsigned(least)));
            v_limit = least ? uint32_t(least + 5) << 23 : 0;
        };

        uint32_t sb = ring, sb_issue = ring + (S::STAGES - 1) * S::STAGE;
        for (int t = 0; t < steps; ++t) {
            const int nx = t + S::STAGES - 1;
            if (nx < steps) {
                if ((nx & 7) == 0) {
                    runs = runs_next;
                    miss_issued = miss_next;
                    runs_next = lookup(nx + 8, &miss_next);
                }
                issue(nx, sb_issue);
            }
            commit();
            if ((t & 7) == 0) miss_now = miss_issued;
            asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 1) : "memory");
            __syncwarp();
            const int key0 = first + t * KV4_STEP;

            // one key a lane: its scales and biases in fp32, and the values' z. A key out of range has none; one whose
            // values are not finite has none either and a NaN for its key, which only the rows that see it meet.
            const uint32_t miss = (miss_now >> ((t & 7) * 4)) & 0xfu;  // runs of 8 keys whose page is missing
            {
                float w[4][GR];  // ks, kb, vs, vb
                const uint32_t p = sb + 2 * S::KV_BYTES + (D == 64 ? lane & ~1 : lane) * S::SC;
                if constexpr (D == 64) {
                    const uint4 v = lds128(p);
                    const int sh = (lane & 1) * 16;
                    w[0][0] = F16Traits<T>::to_f32((v.x >> sh) & 0xffffu), w[1][0] = F16Traits<T>::to_f32((v.y >> sh) & 0xffffu);
                    w[2][0] = F16Traits<T>::to_f32((v.z >> sh) & 0xffffu), w[3][0] = F16Traits<T>::to_f32((v.w >> sh) & 0xffffu);
                } else {
#pragma unroll
                    for (int i = 0; i < GR / 2; ++i) {
                        const uint4 v = lds128(p + 16 * i);
                        const uint32_t x4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // D = 128: one word an array; D = 256: two
                            const int arr = D == 128 ? k : 2 * i + k / 2, g = D == 128 ? 0 : 2 * (k & 1);
                            w[arr][g] = F16Traits<T>::to_f32(x4[k] & 0xffffu);
                            w[arr][g + 1] = F16Traits<T>::to_f32(x4[k] >> 16);
                        }
                    }
                }
                float top = 0.0f, most = 0.0f;
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    top = fmaxf(top, fabsf(w[2][g]));
                    most += fabsf(w[2][g]) + fabsf(w[3][g]);
                }
                const int key = key0 + lane;
                const bool dead = key < lo_min || key >= hi_max || ((miss >> (lane >> 3)) & 1);
                if (dead || !(most < INFINITY)) {
                    top = 0.0f;
#pragma unroll
                    for (int g = 0; g < GR; ++g) w[0][g] = __int_as_float(0x7fffffff), w[2][g] = 0.0f, w[3][g] = 0.0f;
                }
                // the value scales' powers of two: larger scales are met by a smaller one
                const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
                if (bits >= v_limit) fit(bits, top, key0);
                float f[S::FL];
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    // round(-vb / vs) in 0 .. 15, its bits the last of 1.5 * 2^23 + z
                    const float u = fminf(fmaxf(__fdividef(-w[3][g], w[2][g]), 0.0f), 15.0f) + 12582912.0f;
                    f[g] = w[0][g] * 4096.0f;
                    f[GR + g] = w[1][g];
                    f[2 * GR + g] = w[2][g] * vf;
                    f[3 * GR + g] = fmaf(u - 12582912.0f, w[2][g], w[3][g]) * vf;
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(z_at + g * 64), "h"(uint16_t(__float_as_uint(u) & 15u)) : "memory");
                }
#pragma unroll
                for (int i = 0; i < S::FL; i += 4)
                    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(made + (lane * S::FL + i) * 4), "f"(f[i]),
                                 "f"(f[i + 1]), "f"(f[i + 2]), "f"(f[i + 3])
                                 : "memory");
                __syncwarp();
            }

            // scores of this lane's keys (chunk h, half u): key0 + 16 h + 8 u + p8(gid)
            float sc[NT][2][2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float acc[NT][GR][4];
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                    for (int g = 0; g < GR; ++g)
#pragma unroll
                        for (int u = 0; u < 4; ++u) acc[tt][g][u] = 0.0f;
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    const uint32_t p = sb + k_at[g] + h * 16 * S::RB;
                    uint32_t xw[2], yw[2];
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(xw[0]), "=r"(xw[1]) : "r"(p));
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(yw[0]), "=r"(yw[1]) : "r"(p + 8 * S::RB));
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int mm = 0; mm < 2; ++mm) {
                            const uint32_t xs = mm ? xw[u] >> 8 : xw[u], ys = mm ? yw[u] >> 8 : yw[u];
                            const uint32_t a0 = xs & 0x000f000fu, a1 = ys & 0x000f000fu, a2 = xs & 0x00f000f0u, a3 = ys & 0x00f000f0u;
#pragma unroll
                            for (int tt = 0; tt < NT; ++tt)
                                mma_16816<__half>(acc[tt][g], a0, a1, a2, a3, qb[tt][g][u][mm][0], qb[tt][g][u][mm][1]);
                        }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float f[2 * GR];  // ks', kb
                    kv4_floats<2 * GR>(f_at + (16 * h + 8 * u) * S::FL * 4, f);
#pragma unroll
                    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float s = f[GR] * qs[tt][0][e];
#pragma unroll
                            for (int g = 1; g < GR; ++g) s = fmaf(f[GR + g], qs[tt][g][e], s);
#pragma unroll
                            for (int g = 0; g < GR; ++g) s = fmaf(f[g], acc[tt][g][2 * u + e], s);
                            sc[tt][h][u][e] = s * alpha[tt][e];
                        }
                }
            }
            if (partly(key0, miss)) {  // some row does not see some key
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        int lo, hi;
                        column(tt, e, &lo, &hi);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const int key = key0 + 16 * h + 8 * u + kv4_p8(gid);
                                if (key < lo || key >= hi || ((miss >> (2 * h + u)) & 1)) sc[tt][h][u][e] = -INFINITY;
                            }
                    }
            }

            // softmax: the reference m of a column (its 8 lanes agree on it) follows the maximum when that has grown by 2^4
            bool grown = false;
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    grown = grown || fmaxf(fmaxf(sc[tt][0][0][e], sc[tt][0][1][e]), fmaxf(sc[tt][1][0][e], sc[tt][1][1][e])) >
                                         m[tt][e] + 4.0f;
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int tt = 0; tt < NT; ++tt) {
                    float corr[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(fmaxf(sc[tt][0][0][e], sc[tt][0][1][e]), fmaxf(sc[tt][1][0][e], sc[tt][1][1][e]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        mx = fmaxf(mx, m[tt][e]);
                        corr[e] = mx == -INFINITY ? 1.0f : kv4_ex2(m[tt][e] - mx);
                        m[tt][e] = mx;
                        l[tt][e] *= corr[e];
                    }
                    rescale(tt, corr[0], corr[1]);
                }
            }
            uint32_t pb[NT][2][GR][2];
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mz = (m[tt][e] == -INFINITY ? 0.0f : m[tt][e]) - xl[tt][e];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int u = 0; u < 2; ++u) sc[tt][h][u][e] = kv4_ex2(sc[tt][h][u][e] - mz);
                    l[tt][e] += (sc[tt][0][0][e] + sc[tt][0][1][e]) + (sc[tt][1][0][e] + sc[tt][1][1][e]);
                }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float f[2 * GR];  // vs', vb'
                    kv4_floats<2 * GR>(f_at + ((16 * h + 8 * u) * S::FL + 2 * GR) * 4, f);
#pragma unroll
                    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                        for (int g = 0; g < GR; ++g) {
                            hb[tt][g][0] = fmaf(sc[tt][h][u][0], f[GR + g], hb[tt][g][0]);
                            hb[tt][g][1] = fmaf(sc[tt][h][u][1], f[GR + g], hb[tt][g][1]);
                            pb[tt][h][g][u] = kv4_transpose(cvt_f16x2(sc[tt][h][u][1] * f[g], sc[tt][h][u][0] * f[g]));
                        }
                }

            // values: keys p8(2c), p8(2c + 1) (+ 8) of a chunk, dimensions 64 g + 8 gid + i
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    const uint32_t pa = sb + va_at[g] + h * 16 * S::RB, pz = sb + vb_at[g] + h * 16 * S::RB;
                    const uint32_t wa = lds32(pa), wb = lds32(pz), wc = lds32(pa + 8 * S::RB), wd = lds32(pz + 8 * S::RB);
                    uint32_t za, zc;
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(za), "=r"(zc) : "r"(zeds + (g * 2 + h) * 32 + 8 * c));
                    uint32_t ab[2], cd[2];
                    ab[0] = prmt(wa, wb, 0x5410u), ab[1] = prmt(wa, wb, 0x7632u);
                    cd[0] = prmt(wc, wd, 0x5410u), cd[1] = prmt(wc, wd, 0x7632u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t xs = i & 1 ? ab[i >> 1] >> 8 : ab[i >> 1], ys = i & 1 ? cd[i >> 1] >> 8 : cd[i >> 1];
                        const uint32_t a0 = kv4_sub(xs & 0x000f000fu, za), a1 = kv4_sub(xs & 0x00f000f0u, za << 4);
                        const uint32_t a2 = kv4_sub(ys & 0x000f000fu, zc), a3 = kv4_sub(ys & 0x00f000f0u, zc << 4);
#pragma unroll
                        for (int tt = 0; tt < NT; ++tt)
                            mma_16816<__half>(o[tt][4 * g + i], a0, a1, a2, a3, pb[tt][h][g][0], pb[tt][h][g][1]);
                    }
                }
            }
            __syncwarp();
            sb = sb == ring + (S::STAGES - 1) * S::STAGE ? ring : sb + S::STAGE;
            sb_issue = sb_issue == ring + (S::STAGES - 1) * S::STAGE ? ring : sb_issue + S::STAGE;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (CL || x >= x1) grid_dep_launch();

        // ---- the four warps' states joined in shared memory (over the rings) ----
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], d);
#pragma unroll
                    for (int g = 0; g < GR; ++g) hb[t][g][e] += __shfl_xor_sync(0xffffffffu, hb[t][g][e], d);
                }
        __syncthreads();  // every warp is done with its ring
        float* cm = reinterpret_cast<float*>(kv4_smem);  // [warp][R] m, then l, then O [warp][R][D]
        float *cl = cm + KV4_NW * R, *co = cl + KV4_NW * R;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float up = __uint_as_float(uint32_t(127 - int(fmaxf(xl[t][e], 0.0f))) << 23), inv = up / vf;
                const int col = warp * R + 8 * t + 2 * c + e;
                if (gid == 0) cm[col] = m[t][e], cl[col] = l[t][e] * up;
                float* dst = co + col * D + 8 * gid;
#pragma unroll
                for (int g = 0; g < GR; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float2*>(dst + 64 * g + 2 * i) =
                            make_float2(fmaf(o[t][4 * g + i][e], 16777216.0f, hb[t][g][e]) * inv,
                                        fmaf(o[t][4 * g + i][2 + e], 1048576.0f, hb[t][g][e]) * inv);
            }
        __syncthreads();
        const bool whole = !CL && st0 == 0 && st1 == rq.steps();
        float* mine = co + KV4_NW * R * D;  // (CL) this CTA's [R] m, [R] l, [R][D] O
        const size_t part = ((size_t)blockIdx.x * 2 + (st0 == 0 ? 1 : 0)) * R;
        // a warp a row, a lane V neighbouring dimensions at a time
        constexpr int V = D >= 128 ? 4 : 2, VU = D / (32 * V);
        using Vec = std::conditional_t<V == 4, float4, float2>;
        auto put = [&](int j, float M, float L, const float (&O)[VU][V], float sink) {
            const int qi = (row0 + j) / G, head = kvh * G + row0 + j - qi * G;
            uint16_t* dst = a.out + ((size_t)(rq.first + qi) * a.H + head) * D + lane * V;
#pragma unroll
            for (int u = 0; u < VU; ++u) {
                uint32_t h[V / 2];
#pragma unroll
                for (int i = 0; i < V; i += 2)
                    h[i / 2] = kv4_finish<T>(M, L, O[u][i], sink) | uint32_t(kv4_finish<T>(M, L, O[u][i + 1], sink)) << 16;
                if constexpr (V == 4) *reinterpret_cast<uint2*>(dst + u * 32 * V) = make_uint2(h[0], h[1]);
                else *reinterpret_cast<uint32_t*>(dst + u * 32 * V) = h[0];
            }
        };
        for (int j = warp; j < rows; j += KV4_NW) {
            alignas(16) float O[VU][V];
            float M = -INFINITY, L = 0.0f;
            const float sink = kv4_sink(a.sinks, kvh * G + (row0 + j) % G);
#pragma unroll
            for (int u = 0; u < VU; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) O[u][i] = 0.0f;
#pragma unroll
            for (int w = 0; w < KV4_NW; ++w) M = fmaxf(M, cm[w * R + j]);
#pragma unroll
            for (int w = 0; w < KV4_NW; ++w) {
                const float f = cm[w * R + j] == -INFINITY ? 0.0f : kv4_ex2(cm[w * R + j] - M);
                L += cl[w * R + j] * f;  // (a NaN's l has no m: NaN * 0)
#pragma unroll
                for (int u = 0; u < VU; ++u) {
                    alignas(16) float x[V];
                    *reinterpret_cast<Vec*>(x) = *reinterpret_cast<const Vec*>(co + (w * R + j) * D + (u * 32 + lane) * V);
#pragma unroll
                    for (int i = 0; i < V; ++i) O[u][i] += f != 0.0f ? x[i] * f : 0.0f;
                }
            }
            if (whole) {
                put(j, M, L, O, sink);
                continue;
            }
            float* dst = (CL ? mine + 2 * R + j * D : a.part_o + (part + j) * D) + lane * V;
#pragma unroll
            for (int u = 0; u < VU; ++u) *reinterpret_cast<Vec*>(dst + u * 32 * V) = *reinterpret_cast<const Vec*>(O[u]);
            if (CL && lane == 0) mine[j] = M, mine[R + j] = L;
            if (!CL && lane == 0) a.part_ml[2 * (part + j)] = M, a.part_ml[2 * (part + j) + 1] = L;
        }
        if constexpr (CL) {
            cluster_sync();
            const int C = int(kv4_cluster_size());
            const uint32_t base32 = smem_u32(mine);
            for (int j = int(cluster_ctarank()) + C * warp; j < rows; j += C * KV4_NW) {
                const float sink = kv4_sink(a.sinks, kvh * G + (row0 + j) % G);
                const uint32_t own = map_peer(base32 + j * 4, min(lane, C - 1));  // lane k: CTA k's m and l
                const float m = lane < C ? ld_dsmem_f(own) : -INFINITY, l = lane < C ? ld_dsmem_f(own + R * 4) : 0.0f;
                alignas(16) float x[8][VU * V], O[VU][V];
                float M = m;
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int i = 0; i < VU * V; i += V) {
                        const uint32_t at = map_peer(base32, min(k, C - 1)) + (2 * R + j * D + i * 32 + lane * V) * 4;
                        if constexpr (V == 4) {
                            *reinterpret_cast<float4*>(&x[k][i]) = k < C ? ld_dsmem_f4(at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        } else {
#pragma unroll
                            for (int e = 0; e < V; ++e) x[k][i + e] = k < C ? ld_dsmem_f(at + 4 * e) : 0.0f;
                        }
                    }
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
                M = __shfl_sync(0xffffffffu, M, 0);
                const float f = m == -INFINITY ? 0.0f : kv4_ex2(m - M);
                float L = l * f;  // (a NaN's l has no m: NaN * 0)
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
                L = __shfl_sync(0xffffffffu, L, 0);
#pragma unroll
                for (int u = 0; u < VU; ++u)
#pragma unroll
                    for (int i = 0; i < V; ++i) O[u][i] = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
                    for (int u = 0; u < VU; ++u)
#pragma unroll
                        for (int i = 0; i < V; ++i) O[u][i] += fk != 0.0f ? x[k][u * V + i] * fk : 0.0f;
                }
                put(j, M, L, O, sink);
            }
            cluster_sync();  // no CTA leaves while another reads it
        }
        __syncthreads();  // before the next item's ring
    }
}

// One CTA a (share, row): the parts of the item that a share's start divides, joined with the row's sink.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4AttArgs a) {
    constexpr int R = 8 * NT;
    __shared__ float4 sum[4][D / 4];
    __shared__ float4 sml[4];
    grid_dep_wait();
    const int i = blockIdx.x, j = blockIdx.y, warp = threadIdx.x >> 5;
    const int32_t* rec = a.records + i * 8;
    if (!rec[0] || j >= rec[2]) return;
    const int row = rec[5] + j, qi = row / a.G, head = rec[3] * a.G + row - qi * a.G;
    kv4_join_row<T, D, 4>(a, R, j, i - 1, rec[4], warp, kv4_sink(a.sinks, head), a.out + ((size_t)(rec[1] + qi) * a.H + head) * D,
                          sum, sml);
}

// ---- host ----------------------------------------------------------------------------------------

bool kv4_attend_shape_ok(int N, int B, int max_q, int H, int KVH, int width, int window) {
    return N >= 0 && B >= 1 && B <= 65535 && max_q >= 1 && H >= 1 && KVH >= 1 && KVH <= 65535 && H % KVH == 0 &&
           (long long)max_q * (H / KVH) < (1 << 30) && width >= 1 && window >= 0;
}

// One wave of CTAs, as many as are resident.
static int kv4_ctas(int D, int R, int sms) { return sms * kv4_resident(D, R / 8); }

// Rows of kv4_attend's tiles, and the rows up to which a request is its own (above: kv4_prefill). 8 rows, or tiles of 16, if
// every request has at most 64 rows (32 at D = 256, where 16 rows' registers spill), or if all tiles' steps, by the keys that
// the table can name, are no more than 8 a CTA (4 at D = 256); else as many as one query has, 8 or 16, for the requests of a
// mixed batch that only decode. 0: none.
// Each tile unpacks the keys again, but kv4_prefill unpacks slower. 16 requests of 8,192 keys, 4 kv heads, here and there:
// D = 128, 24 rows 66 and 111 us, 48 rows 91 and 118, 64 rows 116 and 123; D = 64, 64 rows 77 and 92; D = 256 (2 kv heads),
// 32 rows 99 and 100, 40 rows 132 and 99. And its items cost more to begin and end. One request, 4 kv heads, D = 128: 128 rows
// on 500 keys 12.5 and 26.6 us, 1,024 rows on 128 keys 12.8 and 33.7; at the limit, 1,024 rows on 2,000 keys, 42.9 and 43.2;
// D = 256 (2 kv heads): 512 rows on 500 keys 22.8 and 36.7.
static void kv4_rows(int max_q, int G, int D, int B, int KVH, long long room, int* R, int* split) {
    const long long most = (long long)max_q * G, own = D == 256 ? 32 : 64;
    const double steps = double((most + 15) / 16) * B * KVH * double((room + KV4_STEP - 1) / KV4_STEP);
    const bool few = most <= own || steps <= (D == 256 ? 4.0 : 8.0) * kv4_ctas(D, 16, device_info().sm_count);
    *R = most <= 8 || (!few && G <= 8) ? 8 : 16;
    *split = few ? int(most) : G <= 16 ? *R : 0;
}

static size_t kv4_few_bytes(int D, int R, int sms) {
    return size_t(kv4_ctas(D, R, sms)) * (2 * R * (2 + D) * sizeof(float) + 8 * sizeof(int32_t));
}

size_t kv4_prefill_workspace_bytes(int D, int sms, int B, int KVH, int G, int max_q, long long room);
bool kv4_prefill_dense(int D, int B, int KVH, int G, int max_q, long long room);
int kv4_prefill_run(const Kv4AttArgs& a, int D, int dtype, void* workspace, cudaStream_t st);

size_t kv4_attend_workspace_bytes(int B, int max_q, int H, int KVH, int D, long long room) {
    int R, split;
    kv4_rows(max_q, H / KVH, D, B, KVH, room, &R, &split);
    const int sms = device_info().sm_count;
    const bool many = (long long)max_q * (H / KVH) > split;
    return (split ? kv4_few_bytes(D, R, sms) : 0) + (many ? kv4_prefill_workspace_bytes(D, sms, B, KVH, H / KVH, max_q, room) : 0);
}

// CTAs a cluster where the clustered form is used, 0 where it is not: as many (up to 8) as leave every item's cluster
// resident at once, if no request can have more than 8 steps a CTA. That spares the second launch and the scan of the
// lengths: one request of 1,001 keys takes 8.5 us, 12.5 with the even split. Beyond, the split is worth more (items differ,
// and steps go to every SM): 4 requests of 131,072 keys leave a cluster form 128 of 444 CTAs.
static int kv4_cluster(int B, int KVH, int split_rows, int max_q, int window, long long room, int D, int R, int sms) {
    const long long items = (long long)B * KVH * ((split_rows + R - 1) / R);
    const long long seen = window ? (room < (long long)window + max_q + KV4_STEP ? room : (long long)window + max_q + KV4_STEP) : room;
    const long long steps = (seen + KV4_STEP - 1) / KV4_STEP;
    int C = 8;
    while (C > 1 && (items * C > kv4_ctas(D, R, sms) || C / 2 >= steps)) C /= 2;
    return items * C <= kv4_ctas(D, R, sms) && steps <= 8 * C ? C : 0;
}

int kv4_attend_forms(int B, int max_q, int H, int KVH, int D, int width, int page, int window) {
    const int G = H / KVH;
    const long long room = (long long)width * page;
    int R, split, forms = 0;
    kv4_rows(max_q, G, D, B, KVH, room, &R, &split);
    if (split) forms |= kv4_cluster(B, KVH, split, max_q, window, room, D, R, device_info().sm_count) ? LQ_KV4_CLUSTERS : LQ_KV4_SPLIT;
    if ((long long)max_q * G > split) forms |= kv4_prefill_dense(D, B, KVH, G, max_q, room) ? LQ_KV4_DENSE : LQ_KV4_TILES;
    return forms;
}

template <typename T, int D, int NT>
static int kv4_attend_n(Kv4AttArgs a, cudaStream_t st) {
    constexpr int R = 8 * NT;
    constexpr size_t merge = size_t(KV4_NW + 1) * R * (2 + D) * sizeof(float);
    constexpr size_t smem = merge > size_t(Kv4Shape<D>::RING) ? merge : size_t(Kv4Shape<D>::RING);
    static std::atomic<uint32_t> set{0}, set_cl{0}, none{0};
    const int sms = device_info().sm_count, n = kv4_ctas(D, R, sms);
    const int C = kv4_cluster(a.B, a.pool.KVH, a.split_rows, a.max_q, a.window, (long long)a.width * a.pool.page, D, R, sms);
    if (C)
        return kv4_launch(kv4_attend_kernel<T, D, NT, true>, set_cl, dim3(a.B * a.pool.KVH * ((a.split_rows + R - 1) / R) * C), dim3(KV4_NW * 32), smem, st, a, C);
    int rc = kv4_launch(kv4_attend_kernel<T, D, NT, false>, set, dim3(n), dim3(KV4_NW * 32), smem, st, a);
    if (rc) return rc;
    return kv4_launch(kv4_join_kernel<T, D, NT>, none, dim3(n, R), dim3(128), 0, st, a);
}

template <typename T, int D>
static int kv4_attend_d(const Kv4AttArgs& a, int R, cudaStream_t st) {
    return R == 8 ? kv4_attend_n<T, D, 1>(a, st) : kv4_attend_n<T, D, 2>(a, st);
}

template <typename T>
static int kv4_attend_t(const Kv4AttArgs& a, int D, int R, cudaStream_t st) {
    return D == 64    ? kv4_attend_d<T, 64>(a, R, st)
           : D == 128 ? kv4_attend_d<T, 128>(a, R, st)
                      : kv4_attend_d<T, 256>(a, R, st);
}

int kv4_attend_run(const Kv4Pool& pool, const void* q, int N, const int32_t* q_start, int max_q, const int32_t* table,
                   int width, const int32_t* lens, int B, const float* sinks, float scale, int window, int H, int D,
                   int dtype, void* workspace, size_t workspace_bytes, void* out, cudaStream_t st) {
    if (N == 0) return LQ_OK;
    if (!workspace || workspace_bytes < kv4_attend_workspace_bytes(B, max_q, H, pool.KVH, D, (long long)width * pool.page)) return LQ_E_ARG;
    const int sms = device_info().sm_count;
    Kv4AttArgs a = {};
    a.pool = pool;
    a.q = static_cast<const uint16_t*>(q);
    a.q_start = q_start;
    a.table = table;
    a.lens = lens;
    a.sinks = sinks;
    a.out = static_cast<uint16_t*>(out);
    a.scale_log2 = scale * KV4_LOG2E;
    a.N = N;
    a.B = B;
    a.H = H;
    a.G = H / pool.KVH;
    a.width = width;
    a.window = window;
    a.max_q = max_q;
    int R;
    kv4_rows(max_q, a.G, D, B, pool.KVH, (long long)width * pool.page, &R, &a.split_rows);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if ((long long)max_q * a.G > a.split_rows) {
        const int rc = kv4_prefill_run(a, D, dtype, ws, st);
        if (rc || !a.split_rows) return rc;
        ws += kv4_prefill_workspace_bytes(D, sms, B, pool.KVH, a.G, max_q, (long long)width * pool.page);
    }
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = a.part_o + size_t(kv4_ctas(D, R, sms)) * 2 * R * D;
    a.records = reinterpret_cast<int32_t*>(a.part_ml + size_t(kv4_ctas(D, R, sms)) * 2 * R * 2);
    return dtype == LQ_BF16 ? kv4_attend_t<__nv_bfloat16>(a, D, R, st) : kv4_attend_t<__half>(a, D, R, st);
}

}  // namespace lq
